// The WKV-7 recurrence over whole sequences with its gradients.
//
// S_t = S_{t-1} diag(d_t) + u_t b_t^T + v_t k_t^T,  u_t = S_{t-1} a_t,  y_t = S_t r_t,  d_t = exp(-exp(w_t)),  S 64 x 64 per head.
// With G_t for the gradient of S_t as all later steps and y_t see it, and h_t = G_t b_t (the gradient of u_t):
//   G_t = (G_{t+1} diag(d_{t+1}) + h_{t+1} a_{t+1}^T) + dy_t r_t^T
//   dr_t = S_t^T dy_t,  dv_t = G_t k_t,  dk_t = G_t^T v_t,  db_t = G_t^T u_t,  da_t = S_{t-1}^T h_t,
//   dd_t[j] = sum_i G_t[i, j] S_{t-1}[i, j],  dw_t = dd_t d_t log d_t.
#include <type_traits>

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

__device__ __forceinline__ int seq_length(const WkvSeq& s, int b) {
    return s.lengths ? min(max(s.lengths[b], 0), s.T) : s.T;
}

// A head's steps 0 .. n - 1 of an array, 64 values each, `step` values apart from the first one at `p` on; all heads' states, `each` of them per
// head.
__device__ __forceinline__ Extent steps_extent(const void* p, int64_t n, int64_t step) {
    const int64_t last = n > 0 ? (n - 1) * step : 0, low = last < 0 ? last : 0;
    return Extent(p ? static_cast<const char*>(p) + 2 * low : nullptr, n > 0 ? (uint64_t)((last < 0 ? -last : last) + 64) * 2 : 0);
}
__device__ __forceinline__ Extent input_extent(const WkvSeq& s, int which, int64_t b, int h, int64_t n) {   // of a sequence of n steps
    return steps_extent(static_cast<const char*>(s.x[which]) + 2 * (b * s.bs[which] + h * 64), n, s.ss[which]);
}
__device__ __forceinline__ Extent states_extent(const float* p, int64_t each) { return Extent(p, (uint64_t)gridDim.x * each * 4096 * sizeof(float)); }

// ---- the forward pass ----------------------------------------------------------------------------------------------------
// A block per head: four warps carry 16 rows of the state each in registers (rows do not meet: the accumulators of one product are the operand of the
// next without leaving the warp), others prepare chunks ahead, each a whole one by itself, in a ring of buffers.
using namespace wkvc;
constexpr int FE_BYTES = (L + 1) * N * 4;   // factors relative to the chunk's end (put_factors)
constexpr int HEAD_BYTES = (int)((sizeof(ChunkHead) + 127) / 128 * 128);
constexpr int FWD_V = FWD_TILES * 2 * TILE, FWD_FE = FWD_V + TILE, FWD_HEAD = FWD_FE + FE_BYTES, FWD_BUF = FWD_HEAD + HEAD_BYTES;
static_assert(8 * FWD_BUF <= 227 * 1024, "shared memory of a block");

// Asks for the rows of a later chunk, 32 bytes a lane. (One bulk request per row takes the warp some 50 cycles each.)
__device__ __forceinline__ void prefetch_steps(const void* x, int64_t at, int64_t step, int n_on, int lane, const Extent& in) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = (lane >> 2) + 8 * i;
        const char* p = static_cast<const char*>(x) + 2 * (at + t * step) + (lane & 3) * 32;
        if (t < n_on && in.holds(p, 32)) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    }
}
__device__ __forceinline__ void prefetch_chunk(const WkvSeq& s, int64_t b, int h, int t0, int n_on, int lane, int n_steps) {
#pragma unroll 1
    for (int i = 0; i < 6; ++i) prefetch_steps(s.x[i], b * s.bs[i] + (int64_t)t0 * s.ss[i] + h * N, s.ss[i], n_on, lane, input_extent(s, i, b, h, n_steps));
}

__device__ __forceinline__ float log2_decay(float w) {   // of exp(-exp(w)); finite (2^-2000 is 0 all the same), but for NaN
    const float d = -expf(w) * 1.4426950408889634f;
    return d < -2000.f ? -2000.f : d;
}
// Asks for one vector of a chunk's steps lo .. hi - 1 (zeros at the others) in a tile's place: a lane has eight columns (c8 = lane & 7) of steps lane
// >> 3, + 4, + 8, + 12, here and when it takes them up again. All vectors of a chunk are on their way at once: one after the other they cost a warp
// 2000 cycles each.
__device__ __forceinline__ void stage_steps(uint32_t tile, const char* p, int64_t step, int lo, int hi, bool there, int lane, const Extent& in) {
    if (!AB_BC(lo >= 0 && lo < hi && hi <= L)) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = (lane >> 3) + 4 * i;
        const char* from = p + (there ? min(max(t, lo), hi - 1) * step : 0);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tile + t * 128 + (((lane & 7) ^ (t & 7)) << 4)), "l"(from),
                     "r"(there && t >= lo && t < hi && in.holds(from, 16) ? 16 : 0) : "memory");
    }
}
__device__ __forceinline__ void staged(uint4* u, uint32_t tile, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = (lane >> 3) + 4 * i;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u[i].x), "=r"(u[i].y), "=r"(u[i].z), "=r"(u[i].w) : "r"(tile + t * 128 + (((lane & 7) ^ (t & 7)) << 4)) : "memory");
    }
}
template <int N_LEFT>
__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N_LEFT) : "memory"); }
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ const char* steps_of(const WkvSeq& s, int which, int64_t b, int h, int t0, int lane) {
    return static_cast<const char*>(s.x[which]) + 2 * (b * s.bs[which] + (int64_t)t0 * s.ss[which] + h * N + 8 * (lane & 7));
}
// The factors of steps lo .. hi - 1 (the others' decays are 1), from the log decays behind fe's first row. fe: [L + 1][N], exp(sum before and
// including the steps up to a row's - end), a row for no step first; fb: [L][N], exp(end - sum); decay: exp(end). In a piece of one step (single) fe
// is 1. Returns whether the chunk is steep, and then, but for a piece, writes nothing.
template <bool PIECE>
__device__ __forceinline__ bool factors_of(int lo, int hi, bool single, float* fe, float* fb, float* decay, int lane) {
    float2 c = make_float2(0.f, 0.f), d[L];
#pragma unroll
    for (int t = 0; t < L; ++t) {
        float2 x = *reinterpret_cast<const float2*>(fe + (t + 1) * N + 2 * lane);
        if (PIECE && (t < lo || t >= hi)) x = make_float2(0.f, 0.f);
        c.x += x.x, c.y += x.y;
        d[t] = c;
    }
    if (!PIECE && __any_sync(0xffffffffu, !(c.x >= -STEEP_LOG2) || !(c.y >= -STEEP_LOG2))) return true;
    const bool one = PIECE && single;
    *reinterpret_cast<float2*>(decay + 2 * lane) = make_float2(ex2_(c.x), ex2_(c.y));
    *reinterpret_cast<float2*>(fe + 2 * lane) = one ? make_float2(1.f, 1.f) : make_float2(ex2_(-c.x), ex2_(-c.y));
#pragma unroll
    for (int t = 0; t < L; ++t) {
        *reinterpret_cast<float2*>(fe + (t + 1) * N + 2 * lane) = one ? make_float2(1.f, 1.f) : make_float2(ex2_(d[t].x - c.x), ex2_(d[t].y - c.y));
        *reinterpret_cast<float2*>(fb + t * N + 2 * lane) = make_float2(ex2_(c.x - d[t].x), ex2_(c.y - d[t].y));
    }
    __syncwarp();
    return false;
}
// From the w of a chunk's n_on steps; true: the chunk is steep, and fe has its log decays.
template <class E>
__device__ __forceinline__ bool put_factors(const uint4* u, int n_on, float* fe, float* fb, float* decay, int lane) {
    const int c8 = lane & 7;
#pragma unroll 1
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = (lane >> 3) + 4 * i;
            const float2 x = raw_pair<E>(half ? u[i].z : u[i].x), y = raw_pair<E>(half ? u[i].w : u[i].y);
            float4 d = make_float4(log2_decay(x.x), log2_decay(x.y), log2_decay(y.x), log2_decay(y.y));
            if (t >= n_on) d = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(fe + (t + 1) * N + 8 * c8 + 4 * half) = d;
        }
    __syncwarp();
    return factors_of<false>(0, L, false, fe, fb, decay, lane);
}
// How many steps of a steep chunk are taken at once: 8, 4, 2 or 1, in pieces from its start on. 1024 steps x 64 heads, decays of 2^-2, 2^-3, 2^-6,
// 2^-17 a step: 0.66, 1.9, 4.3, 9.3 ms forward and 2.2, 7.7, 27, 100 ms backward; 0.14 and 0.41 without a steep chunk. This and the next one are not
// inlined: there they cost every chunk registers (4% forward).
__device__ __noinline__ int steep_steps(const float* fe, int lane) {
    int size = 8;
    for (; size > 1; size >>= 1) {
        bool bad = false;
        float2 sum = make_float2(0.f, 0.f);
        for (int t = 0; t < L; ++t) {
            const float2 x = *reinterpret_cast<const float2*>(fe + (t + 1) * N + 2 * lane);
            sum = t & (size - 1) ? make_float2(sum.x + x.x, sum.y + x.y) : x;
            bad |= !(sum.x >= -STEEP_LOG2) || !(sum.y >= -STEEP_LOG2);
        }
        if (!__any_sync(0xffffffffu, bad)) break;
    }
    return size;
}
__device__ __noinline__ void put_piece(int lo, int hi, bool single, float* fe, float* fb, float* decay, int lane) { factors_of<true>(lo, hi, single, fe, fb, decay, lane); }
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
__device__ __forceinline__ float invert(float* work, Frag& f, float (*v)[4], int lane) {
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

__device__ __forceinline__ Extent upstream_extent(const WkvBackward* g, int64_t b, int h, int64_t n) {
    return g && g->dy ? steps_extent(static_cast<const char*>(g->dy) + 2 * (b * g->dy_batch_stride + h * N), n, g->dy_step_stride) : Extent(nullptr, 0);
}
// Asks for a chunk's vectors: w (in fb's place) ahead of the others, b, k, a and r in the low halves of their tiles, v and dy where one of their
// forms is themselves.
template <class E, bool BWD>
__device__ __forceinline__ void stage_chunk(const WkvSeq& s, const WkvBackward* bwd, int64_t b, int h, int t0, int lo, int hi, bool with_w, uint32_t at, uint32_t v, uint32_t v16, uint32_t fb,
                                            int lane, int n_steps) {
    if (with_w) stage_steps(fb, steps_of(s, 1, b, h, t0, lane), 2 * s.ss[1], lo, hi, true, lane, input_extent(s, 1, b, h, n_steps));
    stage_commit();
#pragma unroll 1
    for (int vec = 0; vec < 4; ++vec) {
        const int which = vec == 0 ? 5 : vec == 1 ? 2 : vec == 2 ? 4 : 0, to = vec == 0 ? T_B : vec == 1 ? T_K : vec == 2 ? T_A : T_R;
        stage_steps(at + to * 2 * TILE + TILE, steps_of(s, which, b, h, t0, lane), 2 * s.ss[which], lo, hi, true, lane, input_extent(s, which, b, h, n_steps));
    }
    constexpr bool OWN = std::is_same<E, __half>::value || !BWD;   // fp16 as it is; bf16 as it is for the sums over rows, else to be converted in place
    stage_steps(OWN ? v : v16, steps_of(s, 3, b, h, t0, lane), 2 * s.ss[3], lo, hi, true, lane, input_extent(s, 3, b, h, n_steps));
    if (BWD) {
        const bool there = bwd->dy != nullptr;
        const int64_t at_dy = there ? b * bwd->dy_batch_stride + (int64_t)t0 * bwd->dy_step_stride + h * N + 8 * (lane & 7) : 0;
        const char* dy = static_cast<const char*>(there ? bwd->dy : s.x[3]) + 2 * at_dy;
        stage_steps(OWN ? v + TILE : v16 + 2 * TILE, dy, there ? 2 * bwd->dy_step_stride : 0, lo, hi, there, lane, upstream_extent(bwd, b, h, n_steps));
    }
    stage_commit();
}

// Prepares a chunk (or a piece of one) that is staged and whose factors are in fe and fb. at: the buffer's tiles; v, dy: where those go, in one fp16
// each (exact down to 2^-27 of the largest); v16, dy16: in bf16. BWD: dy, Q and the tile of a are kept too. The code is kept short, in loops: a warp
// runs through it once per chunk, and unrolled (4000 instructions) it waited for them most of the time (a chunk took it 28000 cycles).
template <class E, bool BWD>
__device__ __forceinline__ void prepare_chunk(uint32_t at, uint32_t v, uint32_t v16, const float* fe, const float* fb, ChunkHead* head, int lane) {
    constexpr int AP = BWD ? T_AP : T_A, VECTORS = BWD ? 6 : 5;
    const uint32_t tA = at + T_A * 2 * TILE, tM = at + T_M * 2 * TILE, tAP = at + AP * 2 * TILE;
    const int c8 = lane & 7, tr = lane >> 3;
    stage_wait<0>();
    // a's and r's factors are at most the first row of fe (2^STEEP_LOG2 or a little more), b's and k's at most 1
    const float2 most = *reinterpret_cast<const float2*>(fe + 2 * lane);
    const int grow_by = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(most.x, most.y), 1.f))) >> 23) + 1;
    const float grow = __int_as_float(min(grow_by, 127 + (int)STEEP_LOG2 + 1) << 23);
    auto up_of = [](float down) { return __uint_as_float((254u << 23) - __float_as_uint(down)); };   // of a power of two
#pragma unroll 1
    for (int vec = 0; vec < VECTORS; ++vec) {   // b, k, a, r, v, dy
        if (!BWD && std::is_same<E, __half>::value && vec == 4) {
            if (lane == 0) head->down_in[4] = 1.f;
            break;
        }
        constexpr bool OWN = std::is_same<E, __half>::value || !BWD;
        uint4 x[4];
        staged(x, vec < 4 ? at + (vec == 0 ? T_B : vec == 1 ? T_K : vec == 2 ? T_A : T_R) * 2 * TILE + TILE : OWN ? v + (vec - 4) * TILE : v16 + (vec - 4) * 2 * TILE, lane);
        Scale sc = {1.f, 1.f};
        if (vec < 4 || std::is_same<E, __nv_bfloat16>::value) {   // (fp16 values are themselves in one fp16)
            uint32_t m = 0;   // the order of non-negative floats is that of their bits
#pragma unroll
            for (int i = 0; i < 4; ++i)
                m = __vmaxu2(__vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)), m);
            const float2 f = raw_pair<E>(m);
            sc = scale_for(warp_top_abs(__uint_as_float(max(__float_as_uint(f.x), __float_as_uint(f.y)))) * (vec == 2 || vec == 3 ? grow : 1.f));   // (a NaN is the largest)
        }
        if (vec < 4) {
            const int which = vec == 0 ? T_B : vec == 1 ? T_K : vec == 2 ? T_A : T_R;
            const float* from = (vec < 2 ? fb : vec == 2 ? fe : fe + N) + 8 * c8;   // (a's are of the sums before its step)
            const uint32_t tile = at + which * 2 * TILE;
            if (lane == 0) head->down[which] = sc.down;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {   // two rows at a time: their loads, their stores
                uint32_t hi4[2][4], lo4[2][4];
                float4 w[2][2];
#pragma unroll
                for (int k = 0; k < 2; ++k) w[k][0] = *reinterpret_cast<const float4*>(from + (tr + 4 * (i + k)) * N), w[k][1] = *reinterpret_cast<const float4*>(from + (tr + 4 * (i + k)) * N + 4);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t raw[4] = {x[i + k].x, x[i + k].y, x[i + k].z, x[i + k].w};
                    const float f[8] = {w[k][0].x, w[k][0].y, w[k][0].z, w[k][0].w, w[k][1].x, w[k][1].y, w[k][1].z, w[k][1].w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float2 e = raw_pair<E>(raw[c]);
                        split(e.x * sc.up * f[2 * c], e.y * sc.up * f[2 * c + 1], hi4[k][c], lo4[k][c]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int t = tr + 4 * (i + k);
                    const uint32_t to = tile + t * 128 + ((c8 ^ (t & 7)) << 4);
                    st128(to, hi4[k]);
                    st128(to + TILE, lo4[k]);
                }
            }
        } else {
            if (lane == 0) head->down_in[vec] = sc.down;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = tr + 4 * i;
                const uint32_t raw[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                const uint32_t to = t * 128 + ((c8 ^ (t & 7)) << 4);
                if (std::is_same<E, __half>::value) {
                    if (BWD) {
                        uint32_t hi4[4], lo4[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 e = raw_pair<E>(raw[c]);
                            split_bf16(e.x, e.y, hi4[c], lo4[c]);
                        }
                        st128(v16 + (vec - 4) * 2 * TILE + to, hi4);
                        st128(v16 + (vec - 4) * 2 * TILE + TILE + to, lo4);
                    }
                } else {
                    uint32_t h4[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float2 e = raw_pair<E>(raw[c]);
                        h4[c] = pack_half(e.x * sc.up, e.y * sc.up);
                    }
                    st128(v + (vec - 4) * TILE + to, h4);
                }
            }
        }
    }
    __syncwarp();
    const int g = lane >> 2, q = lane & 3;
#pragma unroll 1
    for (int m = 0; m < 2; ++m) {   // A_ab and A_ak, A_rb and A_rk
        const int ta = m ? T_R : T_A;
        float c[2][2][4];
        zero2(c[0]), zero2(c[1]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            Frag f, w;
            load_frag(f, at + ta * 2 * TILE, kk * 16, lane, load_a);
            load_frag(w, at + T_B * 2 * TILE, kk * 16, lane, load_b);
            mma3(c[0], f, w);
            load_frag(w, at + T_K * 2 * TILE, kk * 16, lane, load_b);
            mma3(c[1], f, w);
        }
        keep_lower(c[0], head->down[ta], head->down[T_B], m ? 0 : 1, lane);
        keep_lower(c[1], head->down[ta], head->down[T_K], m ? 0 : 1, lane);
        const float d1 = put_block(c[1], tM, (m ? M_RK : M_X) * L, lane);
        if (lane == 0) head->down_m[m ? M_RK : M_X] = d1;
        if (m == 0) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half) *reinterpret_cast<float2*>(head->work + (g + 8 * half) * L + 8 * n + 2 * q) = make_float2(c[0][n][2 * half], c[0][n][2 * half + 1]);
        } else {
            const float d = put_block(c[0], tM, M_RB * L, lane);
            if (lane == 0) head->down_m[M_RB] = d;
        }
    }
    __syncwarp();
    Frag qf;
    float qv[2][4];
    const float down_q = invert(head->work, qf, qv, lane);
    if (BWD) {
        put_acc(qv, at + T_Q * 2 * TILE, 0, up_of(down_q), lane);
        if (lane == 0) head->down[T_Q] = down_q;
    }
    float ap[4][2][4], akp[2][4], top = 0.f;
    zero2(akp);
    {
        Frag f;
        load_frag(f, tM, M_X * L, lane, load_bt);
        mma3(akp, qf, f);
        const float e = head->down_m[M_X];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) akp[n][i] *= down_q * e;
    }
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        Frag f;
        zero2(ap[jj]);
        load_frag(f, tA, jj * 16, lane, load_bt);
        mma3(ap[jj], qf, f);
        top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(acc_top(ap[jj]))));
    }
    const float down_a = head->down[T_A];
    const Scale sa = scale_for(warp_top_abs(top));
    __syncwarp();
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) put_acc(ap[jj], tAP, jj * 16, sa.up, lane);
    const float dak = put_block(akp, tM, M_AK * L, lane);
    if (lane == 0) {
        head->down[AP] = sa.down * down_a * down_q;
        head->down_m[M_AK] = dak;
    }
}

__device__ __forceinline__ void decay_rows(float (*S)[4], const ChunkHead* head, int lane) {
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const float2 d = *reinterpret_cast<const float2*>(head->decay + 8 * n + 2 * (lane & 3));
        S[n][0] *= d.x, S[n][1] *= d.y, S[n][2] *= d.x, S[n][3] *= d.y;
    }
}
__device__ __forceinline__ void row_scales(const float (*S)[4], Scale& s0, Scale& s1) {   // of rows g and g + 8
    float top0 = 0.f, top1 = 0.f;
#pragma unroll
    for (int n = 0; n < 8; n += 2) top0 = fmaxf(top0, row_top(S + n, 0)), top1 = fmaxf(top1, row_top(S + n, 1));
    s0 = scale_for(quad_top_abs(top0)), s1 = scale_for(quad_top_abs(top1));
}
// c = c * (row's down) * d
__device__ __forceinline__ void scale_acc(float (*c)[4], const Scale& s0, const Scale& s1, float d) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = c[n][i] * (i < 2 ? s0.down : s1.down) * d;
}
__device__ __forceinline__ void add_acc(float (*c)[4], const float (*x)[4], float d) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = fmaf(x[n][i], d, c[n][i]);
}
__device__ __forceinline__ void add_acc(float (*c)[4], const float (*x)[4], const Scale& s0, const Scale& s1, float d) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = fmaf(x[n][i] * (i < 2 ? s0.down : s1.down), d, c[n][i]);
}
// c (16 rows x 16 steps) = S times a tile's rows
__device__ __forceinline__ void state_times(float (*c)[4], const float (*S)[4], const Scale& s0, const Scale& s1, uint32_t tile, int lane) {
    zero2(c);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        Frag f, g;
        as_a(f, S + 2 * kk, s0.up, s1.up);
        load_frag(g, tile, kk * 16, lane, load_b);
        mma3(c, f, g);
    }
}

// One chunk for 16 rows of the state: S (accumulators of eight n-tiles) becomes the state after it, y the outputs (rows as m, steps as n).
__device__ __forceinline__ void chunk_rows(float (*S)[4], float (*y)[4], uint32_t at, uint32_t v, int ap, const ChunkHead* head, int i0, int lane) {
    const uint32_t tA = at + ap * 2 * TILE, tR = at + T_R * 2 * TILE, tB = at + T_B * 2 * TILE, tK = at + T_K * 2 * TILE, tM = at + T_M * 2 * TILE;
    const int piece = head->piece;
    float u[2][4];
    Scale s0, s1;
    if (piece) {
        row_scales(S, s0, s1);
        state_times(u, S, s0, s1, tA, lane);
        scale_acc(u, s0, s1, head->down[ap]);
    }
    decay_rows(S, head, lane);
    row_scales(S, s0, s1);
    if (!piece) {
        zero2(u), zero2(y);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            Frag f, g;
            as_a(f, S + 2 * kk, s0.up, s1.up);
            load_frag(g, tA, kk * 16, lane, load_b);
            mma3(u, f, g);
            load_frag(g, tR, kk * 16, lane, load_b);
            mma3(y, f, g);
        }
        scale_acc(u, s0, s1, head->down[ap]);
    } else {
        state_times(y, S, s0, s1, tR, lane);
    }
    scale_acc(y, s0, s1, head->down[T_R]);
    uint32_t fv[4];
    load_at(fv, v, i0, lane);
    const float dv = head->down_in[4];
    float x[2][4];
    Frag g;
    zero2(x);
    load_frag(g, tM, M_AK * L, lane, load_b);
    mma2(x, fv, g);
    add_acc(u, x, dv * head->down_m[M_AK]);
    s0 = scale_for(quad_top_abs(row_top(u, 0))), s1 = scale_for(quad_top_abs(row_top(u, 1)));
    Frag fu;
    as_a(fu, u, s0.up, s1.up);
    zero2(x);
    load_frag(g, tM, M_RB * L, lane, load_b);
    mma3(x, fu, g);
    add_acc(y, x, s0, s1, head->down_m[M_RB]);
    zero2(x);
    load_frag(g, tM, M_RK * L, lane, load_b);
    mma2(x, fv, g);
    add_acc(y, x, dv * head->down_m[M_RK]);
    const float db = head->down[T_B], dk = dv * head->down[T_K];
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        float z[2][4];
        zero2(x), zero2(z);
        load_frag(g, tB, jj * 16, lane, load_bt);
        mma3(x, fu, g);
        load_frag(g, tK, jj * 16, lane, load_bt);
        mma2(z, fv, g);
        add_acc(S + 2 * jj, x, s0, s1, db);
        add_acc(S + 2 * jj, z, dk);
    }
}

template <class E> __device__ __forceinline__ uint32_t pack_pair(float x, float y);
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float x, float y) { return pack_half(x, y); }
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Accumulators (rows i0 .. as m, steps as n) to out[step][row], 64 channels per step and `stride` values between steps, steps lo .. hi - 1 of the
// chunk; zeros from step n_on on.
template <class E>
__device__ __forceinline__ void store_steps(const float (*y)[4], E* out, int64_t stride, int i0, int lo, int hi, int n_on, int lane, const Extent& all) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t p = pack_pair<E>(y[n][2 * half], y[n][2 * half + 1]);
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(p));
            const int t = 8 * n + (lane >> 2);
            uint32_t* to = reinterpret_cast<uint32_t*>(out + t * stride + i0 + 8 * half + 2 * (lane & 3));
            if (t >= lo && t < hi && all.holds(to)) *to = t < n_on ? p : 0u;
        }
}
// a state's rows i0 .. i0 + 15 between accumulators and memory
__device__ __forceinline__ void load_rows(float (*S)[4], const float* from, int i0, int lane, const Extent& states) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float2* p = reinterpret_cast<const float2*>(from + (i0 + (lane >> 2) + 8 * half) * N + 8 * n + 2 * (lane & 3));
            const float2 u = from && states.holds(p) ? *p : make_float2(0.f, 0.f);
            S[n][2 * half] = u.x, S[n][2 * half + 1] = u.y;
        }
}
__device__ __forceinline__ void store_rows(const float (*S)[4], float* to, int i0, int lane, const Extent& states) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float2* p = reinterpret_cast<float2*>(to + (i0 + (lane >> 2) + 8 * half) * N + 8 * n + 2 * (lane & 3));
            if (states.holds(p)) *p = make_float2(S[n][2 * half], S[n][2 * half + 1]);
        }
}

// BUFS chunks under way. Four (two blocks per SM) where there are more heads than SMs; eight, which take an SM's shared memory, where there are not:
// a preparing warp takes 18000 cycles a chunk beside one block's row warps, which take 3800, so that four of them hold these up (1024 steps x 64
// heads 163 us, with eight 153; 2 x 4096 x 32 with states kept 774 and 669).
template <class E, int CHUNK_BUFS>
__global__ void __launch_bounds__((CHUNK_BUFS + 4) * 32, CHUNK_BUFS == 4 ? 2 : 1) wkv_chunk_fwd_kernel(const __grid_constant__ WkvFwd p) {
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
        load_rows(S, s.state ? s.state + (size_t)bh * 4096 : nullptr, i0, lane, states_extent(s.state, 1));
        uint32_t phases = 0;
        bool ok = true;
        for (int n = 0; n < chunks && ok; ++n) {
            const int buf = n % CHUNK_BUFS;
            const uint32_t at = smem_u32(smem) + buf * FWD_BUF;
            const ChunkHead* head = reinterpret_cast<const ChunkHead*>(smem + buf * FWD_BUF + FWD_HEAD);
            if (s.ckpt) store_rows(S, s.ckpt + ((size_t)bh * s.n_chunks + n) * 4096, i0, lane, states_extent(s.ckpt, s.n_chunks));
            for (int more = 1; more && ok;) {
                ok = wait_for(&full[buf], phases >> buf & 1u);
                if (!ok) break;
                phases ^= 1u << buf;
                float o[2][4];
                chunk_rows(S, o, at, at + FWD_V, T_A, head, i0, lane);
                const int lo = head->lo, t0 = head->t0;
                more = head->more;
                store_steps<E>(o, y + t0 * stride, stride, i0, lo, min(head->hi, s.T - t0), n_steps - t0, lane, steps_extent(y, s.T, stride));
                __syncwarp();
                if (lane == 0) mbar_arrive(&vacant[buf]);
            }
        }
        store_rows(S, p.state_out + (size_t)bh * 4096, i0, lane, states_extent(p.state_out, 1));
    } else {
        const int buf = warp - 4;
        const uint32_t at = smem_u32(smem) + buf * FWD_BUF;
        ChunkHead* head = reinterpret_cast<ChunkHead*>(smem + buf * FWD_BUF + FWD_HEAD);
        float *fe = reinterpret_cast<float*>(smem + buf * FWD_BUF + FWD_FE), *fb = reinterpret_cast<float*>(smem + buf * FWD_BUF + T_M * 2 * TILE);   // (fb where T_M comes later)
        int uses = 0;
        bool ok = true;
        for (int n = buf; n < chunks && ok; n += CHUNK_BUFS) {
            const int t0 = n * L, n_on = min(L, n_steps - t0);
            if (n + CHUNK_BUFS < chunks) prefetch_chunk(s, b, h, t0 + CHUNK_BUFS * L, min(L, n_steps - t0 - CHUNK_BUFS * L), lane, n_steps);
            for (int i = 0, pieces = 1; i < pieces; ++i) {
                if (uses > 0) ok = wait_for(&vacant[buf], (uint32_t)(uses - 1) & 1u);
                if (!ok) break;
                ++uses;
                const uint32_t fbs = at + T_M * 2 * TILE;
                stage_chunk<E, false>(s, nullptr, b, h, t0, 0, n_on, true, at, at + FWD_V, 0u, fbs, lane, n_steps);
                uint4 w[4];
                stage_wait<1>();
                staged(w, fbs, lane);
                int lo = 0, hi = n_on, single = 0;
                if (put_factors<E>(w, n_on, fe, fb, head->decay, lane)) {
                    const int size = steep_steps(fe, lane);
                    pieces = (n_on + size - 1) / size, lo = i * size, hi = min(lo + size, n_on), single = size == 1;
                    stage_wait<0>();
                    stage_chunk<E, false>(s, nullptr, b, h, t0, lo, hi, false, at, at + FWD_V, 0u, fbs, lane, n_steps);
                    put_piece(lo, hi, single, fe, fb, head->decay, lane);
                }
                if (lane == 0) head->t0 = t0, head->lo = lo, head->hi = i + 1 < pieces ? hi : L, head->more = i + 1 < pieces, head->piece = single;
                prepare_chunk<E, false>(at, at + FWD_V, 0u, fe, fb, head, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[buf]);
            }
        }
    }
    // steps behind the last chunk
    for (int64_t i = (int64_t)chunks * L * 32 + threadIdx.x; i < (int64_t)s.T * 32; i += (CHUNK_BUFS + 4) * 32)
        if (uint32_t* to = reinterpret_cast<uint32_t*>(y + (i >> 5) * stride + (i & 31) * 2); steps_extent(y, s.T, stride).holds(to)) *to = 0u;
}

// ---- the backward pass -----------------------------------------------------------------------------------------------------
// A block per head goes from the last chunk to the first. Four warps carry 16 rows of the state's gradient each and take the state before each chunk
// from what the forward pass kept; what they make of a chunk (u, h, and both states, as bf16 pairs) crosses in shared memory to four others, which
// have 16 columns each and work out the sums over rows: the gradients of r, a, b, k and the decays. Three warps prepare chunks ahead as in the
// forward pass.
constexpr int BWD_BUFS = 3, BWD_WARPS = 8 + BWD_BUFS;
constexpr int BWD_V = BWD_TILES * 2 * TILE, BWD_DY = BWD_V + TILE, BWD_V16 = BWD_DY + TILE, BWD_DY16 = BWD_V16 + 2 * TILE, BWD_FE = BWD_DY16 + 2 * TILE,
              BWD_FB = BWD_FE + FE_BYTES, BWD_HEAD = BWD_FB + L * N * 4, BWD_BUF = BWD_HEAD + HEAD_BYTES;
// what crosses: states 64 x 64 (bf16, hi and lo), slabs of u and h, the 16 x 16 matrices P (fp16), column sums of G o S_E by row warp
constexpr int BIG = N * N * 2, X_S = 0, X_G = X_S + 2 * BIG, X_U = X_G + 2 * BIG, X_H = X_U + 2 * SLAB, X_P = X_H + 2 * SLAB, X_SUM = X_P + 2 * TILE, X_BYTES = X_SUM + 4 * N * 4;
constexpr int BWD_SMEM = BWD_BUFS * BWD_BUF + X_BYTES;
static_assert(BWD_SMEM <= 227 * 1024, "shared memory of a block");

// the state alone, in pieces of a steep chunk
__device__ __noinline__ void advance_rows(float* S, uint32_t at, const ChunkHead* head, int i0, int lane) {
    float y[2][4];
    chunk_rows(reinterpret_cast<float (*)[4]>(S), y, at, at + BWD_V, T_AP, head, i0, lane);
}
// 16 rows' share of the column sums of G o S (times d, per column): a lane's two columns, 2 lane and 2 lane + 1
__device__ __forceinline__ float2 column_sums(const float (*G)[4], const float (*S)[4], const float* decay, bool with_decay, int lane) {
    float2 p[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) p[n] = make_float2(fmaf(G[n][0], S[n][0], G[n][2] * S[n][2]), fmaf(G[n][1], S[n][1], G[n][3] * S[n][3]));
#pragma unroll
    for (int o = 16, m = 4; m > 0; o >>= 1, m >>= 1) {   // half of what a lane holds goes to the lane that keeps it
        const bool up = lane & o;
#pragma unroll
        for (int n = 0; n < m; ++n) {
            const float2 keep = up ? p[n + m] : p[n], give = up ? p[n] : p[n + m];
            p[n] = make_float2(keep.x + __shfl_xor_sync(0xffffffffu, give.x, o), keep.y + __shfl_xor_sync(0xffffffffu, give.y, o));
        }
    }
    if (with_decay) {
        const float2 d = *reinterpret_cast<const float2*>(decay + 2 * lane);
        p[0].x *= d.x, p[0].y *= d.y;
    }
    return p[0];
}
// Sums over a chunk's steps within the columns of an accumulator fragment (step g in x0, g + 8 in x1): from a step on, and before it
__device__ __forceinline__ void sums_from(float& x0, float& x1, int lane) {
    const int g = lane >> 2;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float a = __shfl_down_sync(0xffffffffu, x0, 4 * o), b = __shfl_down_sync(0xffffffffu, x1, 4 * o);
        if (g + o < 8) x0 += a, x1 += b;
    }
    x0 += __shfl_sync(0xffffffffu, x1, lane & 3);
}
__device__ __forceinline__ void sums_before(float& x0, float& x1, int lane) {
    const int g = lane >> 2;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float a = __shfl_up_sync(0xffffffffu, x0, 4 * o), b = __shfl_up_sync(0xffffffffu, x1, 4 * o);
        if (g >= o) x0 += a, x1 += b;
    }
    const float all0 = __shfl_sync(0xffffffffu, x0, 28 + (lane & 3));
    x0 = __shfl_up_sync(0xffffffffu, x0, 4), x1 = __shfl_up_sync(0xffffffffu, x1, 4);
    if (g == 0) x0 = 0.f, x1 = 0.f;
    x1 += all0;
}
// the values of the step after, of the same column
__device__ __forceinline__ void next_step(float& x0, float& x1, int lane) {
    const int g = lane >> 2;
    const float first1 = __shfl_sync(0xffffffffu, x1, lane & 3);
    x0 = __shfl_down_sync(0xffffffffu, x0, 4), x1 = __shfl_down_sync(0xffffffffu, x1, 4);
    if (g == 7) x0 = first1, x1 = 0.f;
}

template <class E>
__global__ void __launch_bounds__(BWD_WARPS * 32, 1) wkv_chunk_bwd_kernel(const __grid_constant__ WkvBwd p) {
    constexpr bool LO = std::is_same<E, __half>::value;   // inputs take two bf16 values
    extern __shared__ __align__(128) unsigned char smem[];   // BWD_BUFS buffers, then what crosses
    __shared__ uint64_t full[BWD_BUFS], vacant[BWD_BUFS], x_full, x_vacant, p_full;
    __shared__ float p_down[4];
    __shared__ int s_failed;
    const WkvSeq& s = p.s;
    const int bh = blockIdx.x, b = bh / s.H, h = bh - b * s.H;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int n_steps = seq_length(s, b), chunks = (n_steps + L - 1) / L;
    const int64_t stride = (int64_t)s.H * N, base = ((int64_t)b * s.T * s.H + h) * N;   // of the gradients
    unsigned char* cross = smem + BWD_BUFS * BWD_BUF;
    const uint32_t x = smem_u32(cross);
    float* x_sum = reinterpret_cast<float*>(cross + X_SUM);
    if (threadIdx.x == 0) {
        for (int i = 0; i < BWD_BUFS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&vacant[i], 8);
        }
        mbar_init(&x_full, 4);
        mbar_init(&x_vacant, 4);
        mbar_init(&p_full, 4);
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
    auto put_grads = [&](int which, int64_t at, uint32_t two) {   // two values of a gradient
        if (!p.g.dx[which]) return;
        uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<E*>(p.g.dx[which]) + at);
        if (steps_extent(static_cast<E*>(p.g.dx[which]) + base, s.T, stride).holds(to)) *to = two;
    };
    bool ok = true;
    if (warp < 4) {
        const int i0 = warp * 16;
        float G[8][4], S[8][4];
        load_rows(G, p.g.dstate_out ? p.g.dstate_out + (size_t)bh * 4096 : nullptr, i0, lane, states_extent(p.g.dstate_out, 1));
        E* dv_out = p.g.dx[3] ? static_cast<E*>(p.g.dx[3]) + base : nullptr;
        uint32_t phases = 0;
        int items = 0;
        for (int n = chunks - 1, buf = 0; n >= 0 && ok; --n, buf = buf + 1 == BWD_BUFS ? 0 : buf + 1) {
            const uint32_t at = smem_u32(smem) + buf * BWD_BUF;
            const ChunkHead* head = reinterpret_cast<const ChunkHead*>(smem + buf * BWD_BUF + BWD_HEAD);
            const float* before = s.ckpt + ((size_t)bh * s.n_chunks + n) * 4096;
            load_rows(S, before, i0, lane, states_extent(s.ckpt, s.n_chunks));
            for (int more = 1; more && ok;) {
                ok = wait_for(&full[buf], phases >> buf & 1u);
                if (!ok) break;
                phases ^= 1u << buf;
                more = head->more;
                if (head->advance) {
                    float T[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) T[i] = S[i >> 2][i & 3];
                    advance_rows(T, at, head, i0, lane);
#pragma unroll
                    for (int i = 0; i < 32; ++i) S[i >> 2][i & 3] = T[i];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&vacant[buf]);
                    continue;
                }
                const bool piece = head->piece;
                const uint32_t tA = at + T_A * 2 * TILE, tR = at + T_R * 2 * TILE, tB = at + T_B * 2 * TILE, tK = at + T_K * 2 * TILE, tM = at + T_M * 2 * TILE;
                Frag f, w;
                Scale s0, s1;
                float xb[2][4], xk[2][4], z[2][4];
                // G b_E^T and G k_E^T, with dy's part
                row_scales(G, s0, s1);
                zero2(xb), zero2(xk);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    as_a(f, G + 2 * kk, s0.up, s1.up);
                    load_frag(w, tB, kk * 16, lane, load_b);
                    mma3(xb, f, w);
                    load_frag(w, tK, kk * 16, lane, load_b);
                    mma3(xk, f, w);
                }
                scale_acc(xb, s0, s1, head->down[T_B]);
                scale_acc(xk, s0, s1, head->down[T_K]);
                uint32_t fdy[4];
                load_at(fdy, at + BWD_DY, i0, lane);
                const float ddy = head->down_in[5];
                zero2(z);
                load_frag(w, tM, M_RB * L, lane, load_bt);
                mma2(z, fdy, w);
                add_acc(xb, z, ddy * head->down_m[M_RB]);
                zero2(z);
                load_frag(w, tM, M_RK * L, lane, load_bt);
                mma2(z, fdy, w);
                add_acc(xk, z, ddy * head->down_m[M_RK]);
                // h
                s0 = scale_for(quad_top_abs(row_top(xb, 0))), s1 = scale_for(quad_top_abs(row_top(xb, 1)));
                as_a(f, xb, s0.up, s1.up);
                load_frag(w, at + T_Q * 2 * TILE, 0, lane, load_bt);
                zero2(xb);
                mma3(xb, f, w);
                scale_acc(xb, s0, s1, head->down[T_Q]);
                // dv
                Scale h0 = scale_for(quad_top_abs(row_top(xb, 0))), h1 = scale_for(quad_top_abs(row_top(xb, 1)));
                Frag fh;
                as_a(fh, xb, h0.up, h1.up);
                zero2(z);
                load_frag(w, tM, M_X * L, lane, load_bt);
                mma3(z, fh, w);
                add_acc(xk, z, h0, h1, head->down_m[M_X]);
                if (dv_out) store_steps<E>(xk, dv_out + head->t0 * stride, stride, i0, head->lo, min(head->hi, s.T - head->t0), n_steps - head->t0, lane, steps_extent(dv_out, s.T, stride));
                // u
                if (!piece) decay_rows(S, head, lane);
                row_scales(S, s0, s1);
                float u[2][4];
                state_times(u, S, s0, s1, at + T_AP * 2 * TILE, lane);
                scale_acc(u, s0, s1, head->down[T_AP]);
                uint32_t fv[4];
                load_at(fv, at + BWD_V, i0, lane);
                zero2(z);
                load_frag(w, tM, M_AK * L, lane, load_b);
                mma2(z, fv, w);
                add_acc(u, z, head->down_in[4] * head->down_m[M_AK]);
                const float2 gs = column_sums(G, S, head->decay, piece, lane);
                // to the column warps
                if (items > 0) ok = wait_for(&x_vacant, (uint32_t)(items - 1) & 1u);
                if (!ok) break;
                ++items;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t hi, lo;
                        const uint32_t to = i0 * 128 + tile_at(g + 8 * half, 8 * i + 2 * q);
                        split_bf16(S[i][2 * half], S[i][2 * half + 1], hi, lo);
                        st32(x + X_S + to, hi);
                        st32(x + X_S + BIG + to, lo);
                        split_bf16(G[i][2 * half], G[i][2 * half + 1], hi, lo);
                        st32(x + X_G + to, hi);
                        st32(x + X_G + BIG + to, lo);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t hi, lo;
                        const uint32_t to = slab_at(i0 + g + 8 * half, 8 * i + 2 * q);
                        split_bf16(u[i][2 * half], u[i][2 * half + 1], hi, lo);
                        st32(x + X_U + to, hi);
                        st32(x + X_U + SLAB + to, lo);
                        split_bf16(xb[i][2 * half], xb[i][2 * half + 1], hi, lo);
                        st32(x + X_H + to, hi);
                        st32(x + X_H + SLAB + to, lo);
                    }
                *reinterpret_cast<float2*>(x_sum + warp * N + 2 * lane) = gs;
                __syncwarp();
                if (lane == 0) mbar_arrive(&x_full);
                // the gradient of the state before the chunk
                const float dr = ddy * head->down[T_R], da = head->down[T_A];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    float y[2][4];
                    zero2(y), zero2(z);
                    load_frag(w, tR, jj * 16, lane, load_bt);
                    mma2(y, fdy, w);
                    load_frag(w, tA, jj * 16, lane, load_bt);
                    mma3(z, fh, w);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 d = *reinterpret_cast<const float2*>(head->decay + jj * 16 + 8 * i + 2 * q);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float e = c & 1 ? d.y : d.x, a = z[i][c] * (c < 2 ? h0.down : h1.down) * da, r = fmaf(y[i][c], dr, G[2 * jj + i][c]);
                            G[2 * jj + i][c] = piece ? fmaf(r, e, a) : (r + a) * e;
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&vacant[buf]);
                if (more) load_rows(S, before, i0, lane, states_extent(s.ckpt, s.n_chunks));
            }
        }
        if (p.g.dstate) store_rows(G, p.g.dstate + (size_t)bh * 4096, i0, lane, states_extent(p.g.dstate, 1));
    } else if (warp < 8) {
        const int cw = warp - 4, c0 = cw * 16;
        uint32_t phases = 0;
        int items = 0;
        for (int n = chunks - 1, buf = 0; n >= 0 && ok; --n, buf = buf + 1 == BWD_BUFS ? 0 : buf + 1) {
            const uint32_t at = smem_u32(smem) + buf * BWD_BUF;
            const ChunkHead* head = reinterpret_cast<const ChunkHead*>(smem + buf * BWD_BUF + BWD_HEAD);
            const float *fe = reinterpret_cast<const float*>(smem + buf * BWD_BUF + BWD_FE), *fb = reinterpret_cast<const float*>(smem + buf * BWD_BUF + BWD_FB);
            for (int more = 1; more && ok;) {
                ok = wait_for(&full[buf], phases >> buf & 1u);
                if (!ok) break;
                phases ^= 1u << buf;
                more = head->more;
                if (head->advance) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&vacant[buf]);
                    continue;
                }
                const uint32_t tA = at + T_A * 2 * TILE, tR = at + T_R * 2 * TILE, tB = at + T_B * 2 * TILE, tK = at + T_K * 2 * TILE;
                const uint32_t vt = at + BWD_V16, dyt = at + BWD_DY16, P = x + X_P;
                const int t0 = head->t0, lo = head->lo, hi = min(head->hi, s.T - t0), n_on = n_steps - t0;
                const bool piece = head->piece;
                uint32_t raw[5][2][2];   // r, w, k, a, b of this warp's columns
#pragma unroll
                for (int v = 0; v < 5; ++v) {
                    const int which = v < 3 ? v : v + 1;
                    const E* from = static_cast<const E*>(s.x[which]) + b * s.bs[which] + (int64_t)t0 * s.ss[which] + h * N + c0 + 2 * q;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int t = g + 8 * half;
                            const uint32_t* p = reinterpret_cast<const uint32_t*>(from + t * s.ss[which] + 8 * i);
                            raw[v][i][half] = t >= lo && t < min(hi, n_on) && input_extent(s, which, b, h, n_steps).holds(p) ? __ldg(p) : 0u;
                        }
                }
                ok = wait_for(&x_full, (uint32_t)items & 1u);
                if (!ok) break;
                auto input = [&](Frag& f, uint32_t tile, int i, void (*how)(uint32_t*, uint32_t, int, int)) {
                    how(f.hi, tile, i, lane);
                    if (LO) how(f.lo, tile + TILE, i, lane);
                };
                auto slab = [&](Frag& f, uint32_t from, int i, void (*how)(uint32_t*, uint32_t, int, int)) {
                    how(f.hi, from, i, lane);
                    how(f.lo, from + SLAB, i, lane);
                };
                {   // one of the four matrices P: (dy, h) by (u, v)
                    float m[2][4];
                    zero2(m);
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {
                        Frag f, w;
                        if (cw < 2) input(f, dyt, kk * 16, load_a);
                        else slab(f, x + X_H, kk * 16, slab_a);
                        if (cw & 1) input(w, vt, kk * 16, load_b);
                        else slab(w, x + X_U, kk * 16, slab_b);
                        if (cw == 0) mmab<LO, true>(m, f, w);
                        else if (cw == 1) mmab<LO, LO>(m, f, w);
                        else if (cw == 2) mmab<true, true>(m, f, w);
                        else mmab<true, LO>(m, f, w);
                    }
                    keep_lower(m, 1.f, 1.f, cw >> 1, lane);
                    const float d = put_block(m, P, cw * L, lane);
                    if (lane == 0) p_down[cw] = d;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full);
                }
                float dr[2][4], da[2][4], db[2][4], dk[2][4];
                zero2(dr), zero2(da), zero2(db), zero2(dk);
#pragma unroll 1
                for (int kk = 0; kk < 4; ++kk) {
                    Frag f, w;
                    load_bt(w.hi, x + X_S + kk * 2048, c0, lane);
                    load_bt(w.lo, x + X_S + BIG + kk * 2048, c0, lane);
                    input(f, dyt, kk * 16, load_a);
                    mmab<LO, true>(dr, f, w);
                    slab(f, x + X_H, kk * 16, slab_a);
                    mmab<true, true>(da, f, w);
                    load_bt(w.hi, x + X_G + kk * 2048, c0, lane);
                    load_bt(w.lo, x + X_G + BIG + kk * 2048, c0, lane);
                    slab(f, x + X_U, kk * 16, slab_a);
                    mmab<true, true>(db, f, w);
                    input(f, vt, kk * 16, load_a);
                    mmab<LO, true>(dk, f, w);
                }
                ok = wait_for(&p_full, (uint32_t)items & 1u);
                if (!ok) break;
                ++items;
                float pr[2][4], pa[2][4], pb[2][4], pk[2][4];
                zero2(pr), zero2(pa), zero2(pb), zero2(pk);
                auto times = [&](float (*c)[4], int block, const Frag& w, float d, void (*how)(uint32_t*, uint32_t, int, int)) {
                    Frag f;
                    float z[2][4];
                    zero2(z);
                    load_frag(f, P, block * L, lane, how);
                    mma3(z, f, w);
                    add_acc(c, z, d * p_down[block]);
                };
#pragma unroll 1
                for (int i = 0; i < 2; ++i) {
                    Frag w;
                    const float d = head->down[i ? T_K : T_B];
                    load_frag(w, i ? tK : tB, c0, lane, load_bt);
                    times(pr, i, w, d, load_a);
                    times(pa, 2 + i, w, d, load_a);
                }
#pragma unroll 1
                for (int i = 0; i < 2; ++i) {
                    Frag w;
                    const float d = head->down[i ? T_A : T_R];
                    load_frag(w, i ? tA : tR, c0, lane, load_bt);
                    times(pb, 2 * i, w, d, load_at);
                    times(pk, 2 * i + 1, w, d, load_at);
                }
                float2 gs[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    gs[i] = make_float2(0.f, 0.f);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float2 t = *reinterpret_cast<const float2*>(x_sum + r * N + c0 + 8 * i + 2 * q);
                        gs[i].x += t.x, gs[i].y += t.y;
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&x_vacant);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = c0 + 8 * i + 2 * q;
                    const float2 dec = *reinterpret_cast<const float2*>(head->decay + j);
                    float pos[2][2], posa[2][2], flow[2][2], lw[2][2];   // [column][half]
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int t = g + 8 * half;
                        const bool on = t >= lo && t < min(hi, n_on);
                        const float2 fr = *reinterpret_cast<const float2*>(fe + (t + 1) * N + j), fa = *reinterpret_cast<const float2*>(fe + t * N + j);
                        const float2 fi = *reinterpret_cast<const float2*>(fb + t * N + j);
                        const float2 r = raw_pair<E>(raw[0][i][half]), wv = raw_pair<E>(raw[1][i][half]), k = raw_pair<E>(raw[2][i][half]);
                        const float2 a = raw_pair<E>(raw[3][i][half]), bb = raw_pair<E>(raw[4][i][half]);
                        float out[5][2];   // r, w, k, a, b
#pragma unroll
                        for (int cc = 0; cc < 2; ++cc) {
                            const int e = 2 * half + cc;
                            const float er = cc ? fr.y : fr.x, ea = cc ? fa.y : fa.x, ei = cc ? fi.y : fi.x;
                            const float grs = dr[i][e] * (piece ? (cc ? dec.y : dec.x) : er), gr = fmaf(pr[i][e], er, grs), ga = (da[i][e] + pa[i][e]) * ea;
                            const float gbs = db[i][e] * ei, gks = dk[i][e] * ei, gbp = pb[i][e] * ei, gkp = pk[i][e] * ei;
                            const float rv = cc ? r.y : r.x, kv = cc ? k.y : k.x, av = cc ? a.y : a.x, bv = cc ? bb.y : bb.x;
                            out[0][cc] = gr, out[2][cc] = gks + gkp, out[3][cc] = ga, out[4][cc] = gbs + gbp;
                            // (a step's pairs with itself cancel, and a piece has no others: left out, nothing of them is multiplied with a steep log
                            // decay)
                            pos[cc][half] = piece ? rv * grs : fmaf(rv, gr, -fmaf(bv, gbp, kv * gkp));
                            posa[cc][half] = av * ga;
                            flow[cc][half] = fmaf(bv, gbs, kv * gks);
                            lw[cc][half] = on ? log2_decay(cc ? wv.y : wv.x) * 0.6931471805599453f : 0.f;
                        }
                        if (t >= lo && t < hi) {
                            const int64_t to = base + (t0 + t) * stride + j;
                            put_grads(0, to, on ? pack_pair<E>(out[0][0], out[0][1]) : 0u);
                            put_grads(2, to, on ? pack_pair<E>(out[2][0], out[2][1]) : 0u);
                            put_grads(4, to, on ? pack_pair<E>(out[3][0], out[3][1]) : 0u);
                            put_grads(5, to, on ? pack_pair<E>(out[4][0], out[4][1]) : 0u);
                        }
                    }
                    if (p.g.dx[1]) {
#pragma unroll
                        for (int cc = 0; cc < 2; ++cc) {
                            next_step(posa[cc][0], posa[cc][1], lane);
                            pos[cc][0] += posa[cc][0], pos[cc][1] += posa[cc][1];
                            sums_from(pos[cc][0], pos[cc][1], lane);
                            sums_before(flow[cc][0], flow[cc][1], lane);
                        }
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int t = g + 8 * half;
                            const float x0 = (gs[i].x + flow[0][half] + pos[0][half]) * lw[0][half], x1 = (gs[i].y + flow[1][half] + pos[1][half]) * lw[1][half];
                            if (t >= lo && t < hi) put_grads(1, base + (t0 + t) * stride + j, t < n_on ? pack_pair<E>(x0, x1) : 0u);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&vacant[buf]);
            }
        }
    } else {
        const int buf = warp - 8;
        const uint32_t at = smem_u32(smem) + buf * BWD_BUF;
        ChunkHead* head = reinterpret_cast<ChunkHead*>(smem + buf * BWD_BUF + BWD_HEAD);
        float *fe = reinterpret_cast<float*>(smem + buf * BWD_BUF + BWD_FE), *fb = reinterpret_cast<float*>(smem + buf * BWD_BUF + BWD_FB);
        int uses = 0;
        const Extent upstream = upstream_extent(&p.g, b, h, n_steps);
        for (int n = chunks - 1 - buf; n >= 0 && ok; n -= BWD_BUFS) {
            const int t0 = n * L, n_on = min(L, n_steps - t0);
            if (n >= BWD_BUFS) {
                const int t1 = t0 - BWD_BUFS * L;
                prefetch_chunk(s, b, h, t1, L, lane, n_steps);
                if (p.g.dy) prefetch_steps(p.g.dy, b * p.g.dy_batch_stride + (int64_t)t1 * p.g.dy_step_stride + h * N, p.g.dy_step_stride, L, lane, upstream);
                const float* kept = s.ckpt + ((size_t)bh * s.n_chunks + n - BWD_BUFS) * 4096;
                if (lane == 0 && states_extent(s.ckpt, s.n_chunks).holds(kept, 4096)) asm volatile("cp.async.bulk.prefetch.L2.global [%0], 16384;" ::"l"(kept) : "memory");
            }
            // a steep chunk: for each piece from the last one, the pieces before it for the state's sake, and then the piece itself
            for (int i = -1, j = 0, last = 0; !last && ok;) {
                if (uses > 0) ok = wait_for(&vacant[buf], (uint32_t)(uses - 1) & 1u);
                if (!ok) break;
                ++uses;
                const uint32_t fbs = at + BWD_FB;
                stage_chunk<E, true>(s, &p.g, b, h, t0, 0, n_on, true, at, at + BWD_V, at + BWD_V16, fbs, lane, n_steps);
                uint4 w[4];
                stage_wait<1>();
                staged(w, fbs, lane);
                int lo = 0, hi = n_on, single = 0, advance = 0;
                last = 1;
                if (put_factors<E>(w, n_on, fe, fb, head->decay, lane)) {
                    const int size = steep_steps(fe, lane);
                    if (i < 0) i = (n_on - 1) / size;
                    advance = j < i, last = i == 0, single = size == 1;
                    lo = (advance ? j : i) * size, hi = min(lo + size, n_on);
                    if (advance) ++j;
                    else --i, j = 0;
                    stage_wait<0>();
                    stage_chunk<E, true>(s, &p.g, b, h, t0, lo, hi, false, at, at + BWD_V, at + BWD_V16, fbs, lane, n_steps);
                    put_piece(lo, hi, single, fe, fb, head->decay, lane);
                }
                if (lane == 0) head->t0 = t0, head->lo = lo, head->hi = hi == n_on ? L : hi, head->more = !last, head->piece = single, head->advance = advance;
                prepare_chunk<E, true>(at, at + BWD_V, at + BWD_V16, fe, fb, head, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[buf]);
            }
        }
    }
    // steps behind the last chunk
    for (int w = 0; w < 6; ++w)
        if (p.g.dx[w])
            for (int64_t i = (int64_t)chunks * L * 32 + threadIdx.x; i < (int64_t)s.T * 32; i += BWD_WARPS * 32)
                put_grads(w, base + (i >> 5) * stride + (i & 31) * 2, 0u);
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
    static PerDeviceOnce once;
    const DeviceProps* props = nullptr;
    const int c = once.run(&props, [&](const DeviceProps&) -> int {
        for (auto k : {wkv_chunk_fwd_kernel<__half, 4>, wkv_chunk_fwd_kernel<__nv_bfloat16, 4>}) AB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * FWD_BUF));
        for (auto k : {wkv_chunk_fwd_kernel<__half, 8>, wkv_chunk_fwd_kernel<__nv_bfloat16, 8>}) AB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * FWD_BUF));
        return OK;
    });
    if (c != OK) return c;
    const bool f16 = s.dtype == AB_DT_F16;
    if (s.B * s.H > props->n_sm) (f16 ? wkv_chunk_fwd_kernel<__half, 4> : wkv_chunk_fwd_kernel<__nv_bfloat16, 4>)<<<s.B * s.H, 8 * 32, 4 * FWD_BUF, st>>>(p);
    else (f16 ? wkv_chunk_fwd_kernel<__half, 8> : wkv_chunk_fwd_kernel<__nv_bfloat16, 8>)<<<s.B * s.H, 12 * 32, 8 * FWD_BUF, st>>>(p);
    return check_cuda(cudaGetLastError(), "ab_wkv7_seq_fwd");
}

int wkv_train_bwd(const ab_wkv7_seq& s, const WkvBackward& g, cudaStream_t st) {
    WkvBwd p = {seq_of(s), g};
    static PerDeviceOnce once;
    const int c = once.run(nullptr, [&](const DeviceProps&) -> int {
        AB_CUDA(cudaFuncSetAttribute(wkv_chunk_bwd_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, BWD_SMEM));
        AB_CUDA(cudaFuncSetAttribute(wkv_chunk_bwd_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, BWD_SMEM));
        return OK;
    });
    if (c != OK) return c;
    if (s.dtype == AB_DT_F16) wkv_chunk_bwd_kernel<__half><<<s.B * s.H, BWD_WARPS * 32, BWD_SMEM, st>>>(p);
    else wkv_chunk_bwd_kernel<__nv_bfloat16><<<s.B * s.H, BWD_WARPS * 32, BWD_SMEM, st>>>(p);
    return check_cuda(cudaGetLastError(), "ab_wkv7_seq_bwd");
}

}  // namespace ab
