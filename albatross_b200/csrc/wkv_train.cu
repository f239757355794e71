// The WKV-7 recurrence over whole sequences with its gradients.
//
// S_t = S_{t-1} diag(d_t) + u_t b_t^T + v_t k_t^T,  u_t = S_{t-1} a_t,  y_t = S_t r_t,  d_t = exp(-exp(w_t)),  S 64 x 64 per head.
// With G_t for the gradient of S_t as all later steps and y_t see it, and h_t = G_t b_t (the gradient of u_t):
//   G_t = (G_{t+1} diag(d_{t+1}) + h_{t+1} a_{t+1}^T) + dy_t r_t^T
//   dr_t = S_t^T dy_t,  dv_t = G_t k_t,  dk_t = G_t^T v_t,  db_t = G_t^T u_t,  da_t = S_{t-1}^T h_t,
//   dd_t[j] = sum_i G_t[i, j] S_{t-1}[i, j],  dw_t = dd_t d_t log d_t.
#include "wkv_chunk.cuh"

namespace ab {

namespace {

struct WkvSeq {
    const void* x[6];
    int64_t bs[6], ss[6];
    const float* state;
    const int* lengths;
    float* ckpt;
    int T, H, n_chunks;
    unsigned even;   // bit i: every pair of values of x[i] is on a 4-byte boundary; bit 6: of dy
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

// ---- the forward pass ----------------------------------------------------------------------------------------------------
// A block per head: four warps carry 16 rows of the state each in registers (rows do not meet: the accumulators of one product are the operand of the next
// without leaving the warp), four others prepare chunks ahead, each a whole one by itself, in a ring of four buffers.
using namespace wkvc;
constexpr int CHUNK_BUFS = 4, CHUNK_THREADS = (CHUNK_BUFS + 4) * 32;
constexpr int FWD_V = FWD_TILES * 2 * TILE, FWD_HEAD = FWD_V + TILE, FWD_BUF = FWD_HEAD + (int)((sizeof(ChunkHead) + 127) / 128 * 128);

// one vector of a chunk's steps: a lane has columns 2 lane, 2 lane + 1
template <class E>
struct Vec {
    uint32_t raw[L];
    __device__ __forceinline__ void load(const WkvSeq& s, int which, int64_t b, int h, int t0, int n_on, int lane) {
        const E* p = static_cast<const E*>(s.x[which]) + b * s.bs[which] + (int64_t)t0 * s.ss[which] + h * N + 2 * lane;
        const bool even = s.even >> which & 1;
#pragma unroll
        for (int t = 0; t < L; ++t) raw[t] = t < n_on ? load_raw(p + t * s.ss[which], even) : 0u;
    }
    __device__ __forceinline__ float top() const {
        uint32_t m = 0;   // the order of non-negative floats is that of their bits
#pragma unroll
        for (int t = 0; t < L; ++t) m = __vmaxu2(m, raw[t] & 0x7fff7fffu);
        const float2 f = raw_pair<E>(m);
        return warp_top_abs(__uint_as_float(max(__float_as_uint(f.x), __float_as_uint(f.y))));   // (a NaN is the largest)
    }
};
__device__ __forceinline__ uint32_t tile_pair(int t, int lane) { return (uint32_t)(t * 128 + (((lane >> 2) ^ (t & 7)) << 4) + (lane & 3) * 4); }
// asks for the rows of a later chunk
__device__ __forceinline__ void prefetch_chunk(const WkvSeq& s, int64_t b, int h, int t0, int n_on, int lane) {
    const int t = lane & 15;
    if (t >= n_on) return;
#pragma unroll
    for (int i = 0; i < 6; i += 2) {
        const int which = i + (lane >> 4);
        const char* p = static_cast<const char*>(s.x[which]) + 2 * (b * s.bs[which] + (int64_t)(t0 + t) * s.ss[which] + h * N);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    }
}

__device__ __forceinline__ float log2_decay(float w) {   // of exp(-exp(w)); finite (2^-2000 is 0 all the same), but for NaN
    const float d = -expf(w) * 1.4426950408889634f;
    return d < -2000.f ? -2000.f : d;
}
// the log2 decays of a chunk, and whether it is steep
template <class E>
__device__ __forceinline__ bool load_decays(const WkvSeq& s, int64_t b, int h, int t0, int n_on, int lane, float2* lw) {
    Vec<E> w;
    w.load(s, 1, b, h, t0, n_on, lane);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int t = 0; t < L; ++t) {
        const float2 f = raw_pair<E>(w.raw[t]);
        lw[t] = t < n_on ? make_float2(log2_decay(f.x), log2_decay(f.y)) : make_float2(0.f, 0.f);
        sum.x += lw[t].x, sum.y += lw[t].y;
    }
    return __any_sync(0xffffffffu, !(sum.x >= -STEEP_LOG2) || !(sum.y >= -STEEP_LOG2));
}

// Writes raw * 2^(exponent of the step) as hi and lo tiles; returns what its values are to be multiplied with. `head`: the exponents are of the sums before each step
// (a), not after it; `sign` * (sum - from).
template <class E, class X>
__device__ __forceinline__ float put_tile(const Vec<E>& v, const float2* lw, uint32_t tile, int lane, float bound, X exponent) {
    const Scale sc = scale_for(v.top() * bound);
    float2 c = make_float2(0.f, 0.f);
#pragma unroll
    for (int t = 0; t < L; ++t) {
        const float2 before = c;
        c.x += lw[t].x, c.y += lw[t].y;
        const float2 f = raw_pair<E>(v.raw[t]);
        uint32_t hi, lo;
        split(f.x * sc.up * ex2_(exponent(before.x, c.x, 0)), f.y * sc.up * ex2_(exponent(before.y, c.y, 1)), hi, lo);
        st32(tile + tile_pair(t, lane), hi);
        st32(tile + TILE + tile_pair(t, lane), lo);
    }
    return sc.down;
}
__device__ __forceinline__ float acc_top(const float (*c)[4]) {
    float m = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __uint_as_float(max(__float_as_uint(m), __float_as_uint(fabsf(c[n][i]))));
    return m;
}
// two n-tiles of accumulators into a tile, columns c0 .. c0 + 15
__device__ __forceinline__ void put_acc(const float (*c)[4], uint32_t tile, int c0, float up, int lane) {
    const int g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t hi, lo;
            split(c[n][2 * half] * up, c[n][2 * half + 1] * up, hi, lo);
            const uint32_t at = tile_at(g + 8 * half, c0 + 8 * n + 2 * q);
            st32(tile + at, hi);
            st32(tile + TILE + at, lo);
        }
}
__device__ __forceinline__ float put_block(const float (*c)[4], uint32_t tile, int c0, int lane) {
    const Scale sc = scale_for(warp_top_abs(acc_top(c)));
    put_acc(c, tile, c0, sc.up, lane);
    return sc.down;
}
// c *= down, and zeros above the diagonal (strict: on it too); (row t, column s)
__device__ __forceinline__ void keep_lower(float (*c)[4], float down1, float down2, int strict, int lane) {
    const int g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = g + 8 * (i >> 1) - strict >= 8 * n + 2 * q + (i & 1) ? c[n][i] * down1 * down2 : 0.f;
}
__device__ __forceinline__ void load_frag(Frag& f, uint32_t tile, int c0, int lane, void (*how)(uint32_t*, uint32_t, int, int)) {
    how(f.hi, tile, c0, lane);
    how(f.lo, tile + TILE, c0, lane);
}
// Q = (1 - A)^-1 for the strictly lower A in `work` (16 x 16), by columns: x_t = [t = c] + sum_{s < t} A[t, s] x_s. Left in `work`; as an A operand.
__device__ __forceinline__ float invert(float* work, Frag& f, int lane) {
    float x[L];
    const int c = lane & 15;
#pragma unroll
    for (int t = 0; t < L; ++t) {
        float row[L];
#pragma unroll
        for (int s = 0; s < t; s += 4) {
            const float4 u = *reinterpret_cast<const float4*>(work + t * L + s);
            row[s] = u.x, row[s + 1] = u.y, row[s + 2] = u.z, row[s + 3] = u.w;
        }
        float p = t == c ? 1.f : 0.f, q = 0.f;
#pragma unroll
        for (int s = 0; s < t; s += 2) {
            p = fmaf(row[s], x[s], p);
            if (s + 1 < t) q = fmaf(row[s + 1], x[s + 1], q);
        }
        x[t] = p + q;
    }
    __syncwarp();
    if (lane < L)
#pragma unroll
        for (int t = 0; t < L; ++t) work[t * L + c] = x[t];
    __syncwarp();
    const int g = lane >> 2, q = lane & 3;
    float v[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float2 u = *reinterpret_cast<const float2*>(work + (g + 8 * half) * L + 8 * n + 2 * q);
            v[n][2 * half] = u.x, v[n][2 * half + 1] = u.y;
        }
    const Scale sc = scale_for(warp_top_abs(acc_top(v)));
    as_a(f, v, sc.up, sc.up);
    return sc.down;
}

// Prepares steps lo .. hi - 1 of a chunk (of n_on that the sequence has in it); lw: log2 decays, zero at the other steps.
template <class E>
__device__ __forceinline__ void prepare_chunk(const WkvSeq& s, int64_t b, int h, int t0, int lo, int hi, const float2* lw, uint32_t buf, ChunkHead* head, int lane) {
    const uint32_t tA = buf + T_A * 2 * TILE, tR = buf + T_R * 2 * TILE, tB = buf + T_B * 2 * TILE, tK = buf + T_K * 2 * TILE, tM = buf + T_M * 2 * TILE, tV = buf + FWD_V;
    float2 end = make_float2(0.f, 0.f);
#pragma unroll
    for (int t = 0; t < L; ++t) end.x += lw[t].x, end.y += lw[t].y;
    auto load = [&](Vec<E>& v, int which) {
        v.load(s, which, b, h, t0, hi, lane);
        if (lo)
#pragma unroll
            for (int t = 0; t < L; ++t) v.raw[t] = t < lo ? 0u : v.raw[t];
    };
    Vec<E> x;
    float down_b, down_k, down_a, down_r;
    auto to_end = [&](float, float c, int i) { return (i ? end.y : end.x) - c; };                          // of steps 0 .. hi - 1: at most 0
    load(x, 5);
    down_b = put_tile(x, lw, tB, lane, 1.f, to_end);
    load(x, 2);
    down_k = put_tile(x, lw, tK, lane, 1.f, to_end);
    load(x, 3);
#pragma unroll
    for (int t = 0; t < L; ++t) st32(tV + tile_pair(t, lane), x.raw[t]);
    // relative to the end a's and r's factors are at most `grow` (2^STEEP_LOG2); in a piece of one step r's is 1, and a's, which meet nothing, are left as they are
    const bool piece = hi - lo == 1;
    const float grow = piece ? 1.f : ex2_(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(-fminf(end.x, end.y), 0.f)))));
    load(x, 4);
    down_a = put_tile(x, lw, tA, lane, grow, [&](float c, float, int i) { return piece ? 0.f : c - (i ? end.y : end.x); });
    load(x, 0);
    down_r = put_tile(x, lw, tR, lane, grow, [&](float, float c, int i) { return piece ? 0.f : c - (i ? end.y : end.x); });
    __syncwarp();
    {
        float ab[2][4], ak[2][4], rb[2][4], rk[2][4];
        zero2(ab), zero2(ak), zero2(rb), zero2(rk);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            Frag fb, fk, f;
            load_frag(fb, tB, kk * 16, lane, load_b);
            load_frag(fk, tK, kk * 16, lane, load_b);
            load_frag(f, tA, kk * 16, lane, load_a);
            mma3(ab, f, fb);
            mma3(ak, f, fk);
            load_frag(f, tR, kk * 16, lane, load_a);
            mma3(rb, f, fb);
            mma3(rk, f, fk);
        }
        keep_lower(ab, down_a, down_b, 1, lane);
        keep_lower(ak, down_a, down_k, 1, lane);
        keep_lower(rb, down_r, down_b, 0, lane);
        keep_lower(rk, down_r, down_k, 0, lane);
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half) *reinterpret_cast<float2*>(head->work + (g + 8 * half) * L + 8 * n + 2 * q) = make_float2(ab[n][2 * half], ab[n][2 * half + 1]);
        const float dx = put_block(ak, tM, M_X * L, lane), d1 = put_block(rb, tM, M_RB * L, lane), d2 = put_block(rk, tM, M_RK * L, lane);
        if (lane == 0) head->down_m[M_X] = dx, head->down_m[M_RB] = d1, head->down_m[M_RK] = d2;
    }
    __syncwarp();
    // (the tiles relative to the end have been read)
    load(x, 4);
    down_a = put_tile(x, lw, tA, lane, 1.f, [](float c, float, int) { return c; });
    load(x, 0);
    down_r = put_tile(x, lw, tR, lane, 1.f, [](float, float c, int) { return c; });
    Frag q;
    const float down_q = invert(head->work, q, lane);
    float ap[4][2][4], akp[2][4], top = 0.f;
    zero2(akp);
    {
        Frag f;
        load_frag(f, tM, M_X * L, lane, load_bt);
        mma3(akp, q, f);
        const float d = down_q, e = head->down_m[M_X];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) akp[n][i] *= d * e;
    }
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        Frag f;
        zero2(ap[jj]);
        load_frag(f, tA, jj * 16, lane, load_bt);
        mma3(ap[jj], q, f);
        top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(acc_top(ap[jj]))));
    }
    const Scale sa = scale_for(warp_top_abs(top));
    __syncwarp();
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) put_acc(ap[jj], tA, jj * 16, sa.up, lane);
    const float dak = put_block(akp, tM, M_AK * L, lane);
    *reinterpret_cast<float2*>(head->decay + 2 * lane) = make_float2(ex2_(end.x), ex2_(end.y));
    if (lane == 0) {
        head->down[T_A] = sa.down * down_a * down_q;
        head->down[T_R] = down_r;
        head->down[T_B] = down_b;
        head->down[T_K] = down_k;
        head->down_m[M_AK] = dak;
    }
}

// One chunk for 16 rows of the state: S (accumulators of eight n-tiles) becomes the state after it, y the outputs (rows as m, steps as n).
template <class E>
__device__ __forceinline__ void chunk_rows(float (*S)[4], float (*y)[4], uint32_t buf, const ChunkHead* head, int i0, int lane) {
    const uint32_t tA = buf + T_A * 2 * TILE, tR = buf + T_R * 2 * TILE, tB = buf + T_B * 2 * TILE, tK = buf + T_K * 2 * TILE, tM = buf + T_M * 2 * TILE;
    float top0 = 0.f, top1 = 0.f;
#pragma unroll
    for (int n = 0; n < 8; n += 2) top0 = fmaxf(top0, row_top(S + n, 0)), top1 = fmaxf(top1, row_top(S + n, 1));
    const Scale s0 = scale_for(quad_top_abs(top0)), s1 = scale_for(quad_top_abs(top1));
    float u[2][4], ys[2][4];
    zero2(u), zero2(ys);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        Frag f, g;
        as_a(f, S + 2 * kk, s0.up, s1.up);
        load_frag(g, tA, kk * 16, lane, load_b);
        mma3(u, f, g);
        load_frag(g, tR, kk * 16, lane, load_b);
        mma3(ys, f, g);
    }
    float v[2][4], acc[2][4];
    load_vt<E>(v, buf + FWD_V, i0, lane);
    const float tv0 = quad_top_abs(row_top(v, 0)), tv1 = quad_top_abs(row_top(v, 1));
    const Scale v0 = scale_for(tv0), v1 = scale_for(tv1);
    uint32_t fv[4];
    as_a_exact(fv, v, v0.up, v1.up);
    zero2(acc);
    {
        Frag g;
        load_frag(g, tM, M_AK * L, lane, load_b);
        mma2(acc, fv, g);
    }
    {
        const float da = head->down[T_A], dr = head->down[T_R], dk = head->down_m[M_AK];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ds = i < 2 ? s0.down : s1.down, dv = i < 2 ? v0.down : v1.down;
                u[n][i] = fmaf(acc[n][i] * dv, dk, u[n][i] * ds * da);
                ys[n][i] = ys[n][i] * ds * dr;
            }
    }
    const float tu0 = quad_top_abs(row_top(u, 0)), tu1 = quad_top_abs(row_top(u, 1));
    // u and v with one scale per row for a product with b's and k's side, whose own scales (powers of two) go to u's and v's
    auto pair = [&](Frag& fu, uint32_t* fv_, float db, float dk, Scale& r0, Scale& r1) {
        r0 = scale_for(fmaxf(tu0 * db, tv0 * dk)), r1 = scale_for(fmaxf(tu1 * db, tv1 * dk));
        as_a(fu, u, db * r0.up, db * r1.up);
        as_a_exact(fv_, v, dk * r0.up, dk * r1.up);
    };
    Frag fu;
    Scale r0, r1;
    pair(fu, fv, head->down_m[M_RB], head->down_m[M_RK], r0, r1);
    zero2(acc);
    {
        Frag g;
        load_frag(g, tM, M_RB * L, lane, load_b);
        mma3(acc, fu, g);
        load_frag(g, tM, M_RK * L, lane, load_b);
        mma2(acc, fv, g);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[n][i] = fmaf(acc[n][i], i < 2 ? r0.down : r1.down, ys[n][i]);
    pair(fu, fv, head->down[T_B], head->down[T_K], r0, r1);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        Frag g;
        zero2(acc);
        load_frag(g, tB, jj * 16, lane, load_bt);
        mma3(acc, fu, g);
        load_frag(g, tK, jj * 16, lane, load_bt);
        mma2(acc, fv, g);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float2 d = *reinterpret_cast<const float2*>(head->decay + jj * 16 + 8 * n + 2 * (lane & 3));
#pragma unroll
            for (int i = 0; i < 4; ++i) S[2 * jj + n][i] = fmaf(acc[n][i], i < 2 ? r0.down : r1.down, S[2 * jj + n][i] * (i & 1 ? d.y : d.x));
        }
    }
}

template <class E> __device__ __forceinline__ uint32_t pack_pair(float x, float y);
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float x, float y) { return pack_half(x, y); }
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Accumulators (rows i0 .. as m, steps as n) to out[step][row], 64 channels per step and `stride` values between steps, steps lo .. hi - 1 of the chunk; zeros
// from step n_on on.
template <class E>
__device__ __forceinline__ void store_steps(const float (*y)[4], E* out, int64_t stride, int i0, int lo, int hi, int n_on, int lane) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t p = pack_pair<E>(y[n][2 * half], y[n][2 * half + 1]);
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(p));
            const int t = 8 * n + (lane >> 2);
            if (t >= lo && t < hi) *reinterpret_cast<uint32_t*>(out + t * stride + i0 + 8 * half + 2 * (lane & 3)) = t < n_on ? p : 0u;
        }
}
// a state's rows i0 .. i0 + 15 between accumulators and memory
__device__ __forceinline__ void load_rows(float (*S)[4], const float* from, int i0, int lane) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float2 u = from ? *reinterpret_cast<const float2*>(from + (i0 + (lane >> 2) + 8 * half) * N + 8 * n + 2 * (lane & 3)) : make_float2(0.f, 0.f);
            S[n][2 * half] = u.x, S[n][2 * half + 1] = u.y;
        }
}
__device__ __forceinline__ void store_rows(const float (*S)[4], float* to, int i0, int lane) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half)
            *reinterpret_cast<float2*>(to + (i0 + (lane >> 2) + 8 * half) * N + 8 * n + 2 * (lane & 3)) = make_float2(S[n][2 * half], S[n][2 * half + 1]);
}

template <class E>
__global__ void __launch_bounds__(CHUNK_THREADS, 2) wkv_chunk_fwd_kernel(const __grid_constant__ WkvFwd p) {
    extern __shared__ __align__(128) unsigned char smem[];   // CHUNK_BUFS buffers
    __shared__ uint64_t full[CHUNK_BUFS], vacant[CHUNK_BUFS];
    __shared__ int s_failed;
    const WkvSeq& s = p.s;
    const int bh = blockIdx.x, b = bh / s.H, h = bh - b * s.H;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_steps = seq_length(s, b), chunks = (n_steps + L - 1) / L;
    if (threadIdx.x == 0) {
        for (int i = 0; i < CHUNK_BUFS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&vacant[i], 4);
        }
        fence_mbar_init();
        s_failed = 0;
    }
    __syncthreads();
    // after the first wait that runs out nobody waits any more
    auto wait_for = [&](uint64_t* bar, uint32_t parity) {
        bool ok = mbar_try_wait(bar, parity);
        if (!ok && !*reinterpret_cast<volatile int*>(&s_failed)) {
            ok = mbar_wait_bounded(bar, parity, 1u << 18);
            if (!ok) {
                *reinterpret_cast<volatile int*>(&s_failed) = 1;
                atomicOr(&g_device_status, DEV_WAIT_HEAD);
            }
        }
        return __all_sync(0xffffffffu, ok) != 0;
    };
    E* y = static_cast<E*>(p.y) + ((int64_t)b * s.T * s.H + h) * N;
    const int64_t stride = (int64_t)s.H * N;
    if (warp < 4) {
        const int i0 = warp * 16;
        float S[8][4];
        load_rows(S, s.state ? s.state + (size_t)bh * 4096 : nullptr, i0, lane);
        uint32_t phases = 0;
        bool ok = true;
        for (int n = 0; n < chunks && ok; ++n) {
            const int buf = n % CHUNK_BUFS;
            const uint32_t at = smem_u32(smem) + buf * FWD_BUF;
            const ChunkHead* head = reinterpret_cast<const ChunkHead*>(smem + buf * FWD_BUF + FWD_HEAD);
            if (s.ckpt) store_rows(S, s.ckpt + ((size_t)bh * s.n_chunks + n) * 4096, i0, lane);
            for (int more = 1; more && ok;) {
                ok = wait_for(&full[buf], phases >> buf & 1u);
                if (!ok) break;
                phases ^= 1u << buf;
                float o[2][4];
                chunk_rows<E>(S, o, at, head, i0, lane);
                const int lo = head->lo, t0 = head->t0;
                more = head->more;
                store_steps<E>(o, y + t0 * stride, stride, i0, lo, min(head->hi, s.T - t0), n_steps - t0, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(&vacant[buf]);
            }
        }
        store_rows(S, p.state_out + (size_t)bh * 4096, i0, lane);
    } else {
        const int buf = warp - 4;
        const uint32_t at = smem_u32(smem) + buf * FWD_BUF;
        ChunkHead* head = reinterpret_cast<ChunkHead*>(smem + buf * FWD_BUF + FWD_HEAD);
        int uses = 0;
        bool ok = true;
        for (int n = buf; n < chunks && ok; n += CHUNK_BUFS) {
            const int t0 = n * L, n_on = min(L, n_steps - t0);
            float2 lw[L];
            const bool steep = load_decays<E>(s, b, h, t0, n_on, lane, lw);
            if (n + CHUNK_BUFS < chunks) prefetch_chunk(s, b, h, t0 + CHUNK_BUFS * L, min(L, n_steps - t0 - CHUNK_BUFS * L), lane);
            const int pieces = steep ? n_on : 1;
            for (int i = 0; i < pieces; ++i) {
                if (uses > 0) ok = wait_for(&vacant[buf], (uint32_t)(uses - 1) & 1u);
                if (!ok) break;
                ++uses;
                const int lo = steep ? i : 0, hi = steep ? i + 1 : n_on;
                if (steep) {
                    float2 one[L];
#pragma unroll
                    for (int t = 0; t < L; ++t) one[t] = t == i ? lw[t] : make_float2(0.f, 0.f);
                    prepare_chunk<E>(s, b, h, t0, lo, hi, one, at, head, lane);
                } else {
                    prepare_chunk<E>(s, b, h, t0, lo, hi, lw, at, head, lane);
                }
                if (lane == 0) head->t0 = t0, head->lo = lo, head->hi = i + 1 < pieces ? hi : L, head->more = i + 1 < pieces;
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[buf]);
            }
        }
    }
    // steps behind the last chunk
    for (int64_t i = (int64_t)chunks * L * 32 + threadIdx.x; i < (int64_t)s.T * 32; i += CHUNK_THREADS)
        *reinterpret_cast<uint32_t*>(y + (i >> 5) * stride + (i & 31) * 2) = 0u;
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
        if (reinterpret_cast<uintptr_t>(s.x[i]) % 4 == 0 && s.batch_stride[i] % 2 == 0 && s.step_stride[i] % 2 == 0) q.even |= 1u << i;
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
    static PerDeviceOnce once;
    const int c = once.run(nullptr, [&](const DeviceProps&) -> int {
        AB_CUDA(cudaFuncSetAttribute(wkv_chunk_fwd_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, CHUNK_BUFS * FWD_BUF));
        AB_CUDA(cudaFuncSetAttribute(wkv_chunk_fwd_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, CHUNK_BUFS * FWD_BUF));
        return OK;
    });
    if (c != OK) return c;
    if (s.dtype == AB_DT_F16) wkv_chunk_fwd_kernel<__half><<<s.B * s.H, CHUNK_THREADS, CHUNK_BUFS * FWD_BUF, st>>>(p);
    else wkv_chunk_fwd_kernel<__nv_bfloat16><<<s.B * s.H, CHUNK_THREADS, CHUNK_BUFS * FWD_BUF, st>>>(p);
    return check_cuda(cudaGetLastError(), "ab_wkv7_seq_fwd");
}

int wkv_train_bwd(const ab_wkv7_seq& s, const WkvBackward& g, cudaStream_t st) {
    WkvBwd p = {seq_of(s), g};
    if (s.dtype == AB_DT_F16) wkv_steps_bwd_kernel<__half><<<s.B * s.H, WT, 0, st>>>(p);
    else wkv_steps_bwd_kernel<__nv_bfloat16><<<s.B * s.H, WT, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), "ab_wkv7_seq_bwd");
}

}  // namespace ab
