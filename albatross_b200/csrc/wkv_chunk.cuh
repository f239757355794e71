// The WKV-7 recurrence in chunks of 16 steps, on the tensor cores: what the forward and the backward kernel share.
//
// Within a chunk, with cw_t the sums of log decays from its start, `end` the whole sum, and everything taken relative to the chunk's end:
//   a_E = a exp(cw_{t-1} - end),  r_E = r exp(cw_t - end),  b_E = b exp(end - cw_t),  k_E = k exp(end - cw_t),  S_E = S diag(exp(end))
//   A_ab = tril(a_E b_E^T, -1),  A_ak = tril(a_E k_E^T, -1),  A_rb = tril(r_E b_E^T),  A_rk = tril(r_E k_E^T)        16 x 16
//   Q = (1 - A_ab)^-1,  a' = Q a_E,  A' = Q A_ak
//   u^T = S_E a'^T + v^T A'^T,   y^T = S_E r_E^T + u^T A_rb^T + v^T A_rk^T,   S <- S_E + u^T b_E + v^T k_E
// (the triangular form of the delta rule's chunks, Yang et al., "Parallelizing linear transformers with the delta rule over sequence length", 2024,
// here for a decay per channel and separate a and b). Backwards, with G the gradient of the state after the chunk, h of u:
//   h^T = (dy^T A_rb + G b_E^T) Q,   dv^T = dy^T A_rk + G k_E^T + h^T A_ak,   G <- (G + dy^T r_E + h^T a_E) diag(exp(end))
//   P_yu = tril(dy u^T),  P_yv = tril(dy v^T),  P_hu = tril(h u^T, -1),  P_hv = tril(h v^T, -1)                       16 x 16
//   dr = (dy S_E + P_yu b_E + P_yv k_E) exp(cw_t - end),   da = (h S_E + P_hu b_E + P_hv k_E) exp(cw_{t-1} - end)
//   db = (u G + P_yu^T r_E + P_hu^T a_E) exp(end - cw_t),   dk = (v G + P_yv^T r_E + P_hv^T a_E) exp(end - cw_t)
// and the gradient of a step's log decay collects what flows through it: from the state before to the state after the chunk (the column sums of G o
// S_E), from steps before it to the state after (b, k times their G parts), from the state before to steps from it on (r, a times their S parts), and
// between steps on both sides (r, a times their P parts less b, k times theirs, summed from it on).
//
// Precision. States and sums are 32-bit. A factor of a product that meets a state is the sum of two fp16 values, hi + lo (22 bits), after scaling by
// a power of two that brings the largest value of its tile (of its row, for states) to 2^13 .. 2^14; three of the four partial products are made, the
// fourth is 2^-22 of the result. v and dy are held in one fp16 value (fp16: as they are; bf16: exact down to 2^-27 of the largest). One product
// therefore costs three (two) mma.sync.m16n8k16; tf32 with its own three would cost six of the same rate. What only ends in 16-bit gradients and sums
// over the rows of a state is split into two bf16 values instead (16 bits, no scale to agree on among warps).
//
// Factors relative to the end grow as the decays shrink: up to exp(-end). Up to 2^16 (decays of 0.5 per step; the model's are above 0.545) the
// split's 22 bits stand, since a tile's values down to 2^-16 of its largest keep them. A chunk beyond that ("steep") is taken in pieces of 8, 4, 2 or
// 1 steps: the same code, with the other steps' inputs as zeros and their decays as ones. In a piece of one step (whose decay may be anything) r_E =
// r, b_E = b, k_E = k, there is no A_ab and A_ak, and u = S a with the state before its decay. Backwards the state before each piece is made again
// from the one before the chunk.
#pragma once
#include "train.cuh"

namespace ab {

namespace wkvc {

constexpr int L = WKV_CHUNK, N = 64;
constexpr float STEEP_LOG2 = 16.f;

// ---- tiles: 16 x 64 fp16, rows of 128 bytes, 16-byte groups exchanged by the row's low bits --------------------------------
constexpr int TILE = L * N * 2;   // bytes
__device__ __forceinline__ uint32_t tile_at(int row, int col) { return (uint32_t)(row * 128 + (((col >> 3) ^ (row & 7)) << 4) + (col & 7) * 2); }
__device__ __forceinline__ void ldsm(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// The four 8 x 8 matrices of 16 rows and columns c0 .. c0 + 15, in the three orders that fragments want:
// rows as n, columns as k (B): registers 0, 1 for n 0..7, 2, 3 for n 8..15
__device__ __forceinline__ void load_b(uint32_t* r, uint32_t tile, int c0, int lane) { ldsm(r, tile + tile_at((lane & 7) + ((lane >> 4) << 3), c0 + ((lane >> 3) & 1) * 8)); }
// rows as m, columns as k (A)
__device__ __forceinline__ void load_a(uint32_t* r, uint32_t tile, int c0, int lane) { ldsm(r, tile + tile_at((lane & 7) + ((lane >> 3) & 1) * 8, c0 + (lane >> 4) * 8)); }
// rows as k, columns as n (B): registers 0, 1 for columns c0 .. c0 + 7, 2, 3 for the next eight
__device__ __forceinline__ void load_bt(uint32_t* r, uint32_t tile, int c0, int lane) { ldsm_t(r, tile + tile_at((lane & 7) + ((lane >> 3) & 1) * 8, c0 + (lane >> 4) * 8)); }
// rows as k, columns as m (A)
__device__ __forceinline__ void load_at(uint32_t* r, uint32_t tile, int c0, int lane) { ldsm_t(r, tile + tile_at((lane & 7) + (lane >> 4) * 8, c0 + ((lane >> 3) & 1) * 8)); }

__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
struct Frag {      // of 16 x 16 values: as A, or as B for two n-tiles
    uint32_t hi[4], lo[4];
};
// c[0], c[1] += a * (two n-tiles of b), three partial products
__device__ __forceinline__ void mma3(float (*c)[4], const Frag& a, const Frag& b) {
#pragma unroll
    for (int n = 0; n < 2; ++n) mma(c[n], a.hi, b.hi[2 * n], b.hi[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma(c[n], a.hi, b.lo[2 * n], b.lo[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma(c[n], a.lo, b.hi[2 * n], b.hi[2 * n + 1]);
}
// the same where a is exact in its high half
__device__ __forceinline__ void mma2(float (*c)[4], const uint32_t* a, const Frag& b) {
#pragma unroll
    for (int n = 0; n < 2; ++n) mma(c[n], a, b.hi[2 * n], b.hi[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma(c[n], a, b.lo[2 * n], b.lo[2 * n + 1]);
}
__device__ __forceinline__ void zero2(float (*c)[4]) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = 0.f;
}

// ---- scales and splits -----------------------------------------------------------------------------------------------------
struct Scale {
    float up, down;   // powers of two, up * down = 1
};
__device__ __forceinline__ Scale scale_for(float top) {   // brings `top` (>= 0) to 2^13 .. 2^14; of 0, infinities and NaN it makes nothing else
    const int e = min(max((__float_as_int(top) >> 23) & 255, 20), 253);
    return {__int_as_float((267 - e) << 23), __int_as_float((e - 13) << 23)};
}
__device__ __forceinline__ float warp_top_abs(float v) {   // largest of non-negative values of a warp; NaN wins
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
__device__ __forceinline__ float quad_top_abs(float v) {   // of the four lanes that share a row of a fragment
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ uint32_t pack_half(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_half(x - f.x, y - f.y);
}
__device__ __forceinline__ float ex2_(float x) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    return e;
}
__device__ __forceinline__ void st128(uint32_t addr, const uint32_t* v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// An accumulator (two n-tiles of 16 rows) as the A operand of a product over its columns, with a scale per row (row g, row g + 8)
__device__ __forceinline__ void as_a(Frag& f, const float (*c)[4], float up0, float up1) {
    split(c[0][0] * up0, c[0][1] * up0, f.hi[0], f.lo[0]);
    split(c[0][2] * up1, c[0][3] * up1, f.hi[1], f.lo[1]);
    split(c[1][0] * up0, c[1][1] * up0, f.hi[2], f.lo[2]);
    split(c[1][2] * up1, c[1][3] * up1, f.hi[3], f.lo[3]);
}
__device__ __forceinline__ float row_top(const float (*c)[4], int half) {   // largest of a row's four values in two n-tiles; half 0: row g, 1: row g + 8
    return fmaxf(fmaxf(fabsf(c[0][2 * half]), fabsf(c[0][2 * half + 1])), fmaxf(fabsf(c[1][2 * half]), fabsf(c[1][2 * half + 1])));
}

// two neighbouring values of an input as floats
template <class E> __device__ __forceinline__ float2 raw_pair(uint32_t u);
template <> __device__ __forceinline__ float2 raw_pair<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <> __device__ __forceinline__ float2 raw_pair<__nv_bfloat16>(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }

// ---- a chunk as the working warps find it --------------------------------------------------------------------------------------
// tiles (hi, then lo); the forward pass has a' in T_A's place
enum { T_A, T_R, T_B, T_K, T_M, FWD_TILES, T_AP = FWD_TILES, T_Q, BWD_TILES };
enum { M_AK, M_RB, M_RK, M_X };                // 16 x 16 matrices side by side in T_M: A', A_rb, A_rk, A_ak
struct ChunkHead {
    float down[BWD_TILES], down_m[4], down_in[6];   // of tiles, of the matrices in T_M, of b, k, a, r, v, dy as they come
    int t0, lo, hi, more;                      // steps t0 + lo .. t0 + hi - 1 of the sequence; more: the chunk goes on in this buffer
    int piece, advance;                        // piece: one step of a steep chunk; advance: the state alone moves on (backward pass)
    alignas(16) float decay[N];                // exp(end)
    alignas(16) float work[L * L];             // the preparing warp's own
};

// ---- bf16 pairs ----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack_bf16(x, y);
    lo = pack_bf16(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// partial products: LA, LB: whether a and b have low halves
template <bool LA, bool LB>
__device__ __forceinline__ void mmab(float (*c)[4], const Frag& a, const Frag& b) {
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_bf16(c[n], a.hi, b.hi[2 * n], b.hi[2 * n + 1]);
    if (LB)
#pragma unroll
        for (int n = 0; n < 2; ++n) mma_bf16(c[n], a.hi, b.lo[2 * n], b.lo[2 * n + 1]);
    if (LA)
#pragma unroll
        for (int n = 0; n < 2; ++n) mma_bf16(c[n], a.lo, b.hi[2 * n], b.hi[2 * n + 1]);
}
// A matrix of 64 rows (channels) x 16 steps, rows of 32 bytes
constexpr int SLAB = N * L * 2;
__device__ __forceinline__ uint32_t slab_at(int row, int t) { return (uint32_t)(row * 32 + (((t >> 3) ^ (row >> 2 & 1)) << 4) + (t & 7) * 2); }
// 16 of its rows as k, steps as m (A)
__device__ __forceinline__ void slab_a(uint32_t* r, uint32_t slab, int i0, int lane) { ldsm_t(r, slab + slab_at(i0 + (lane & 7) + (lane >> 4) * 8, ((lane >> 3) & 1) * 8)); }
// 16 of its rows as k, steps as n (B)
__device__ __forceinline__ void slab_b(uint32_t* r, uint32_t slab, int i0, int lane) { ldsm_t(r, slab + slab_at(i0 + (lane & 7) + ((lane >> 3) & 1) * 8, (lane >> 4) * 8)); }

}  // namespace wkvc
}  // namespace ab
