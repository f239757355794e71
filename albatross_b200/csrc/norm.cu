// Layer norm (in groups: the norm of each head behind the recurrence) and its gradients.
//
// With xh = (x - mean) rstd over a group of m values, y = xh w + b, and e = dy w:
//   dx = rstd (e - mean(e) - xh mean(e xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy.
#include <algorithm>
#include <type_traits>

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

// the arrays of a call
template <class E>
__device__ __forceinline__ Extent x_extent(const NormArgs& a) { return rows_extent(a.x, a.rows, a.x_stride, a.C, sizeof(E)); }
template <class E>
__device__ __forceinline__ Extent dy_extent(const NormArgs& a) { return rows_extent(a.dy, a.rows, a.dy_stride, a.C, sizeof(E)); }
template <class E>
__device__ __forceinline__ Extent dense_extent(const NormArgs& a, const void* p) { return rows_extent(p, a.rows, a.C, a.C, sizeof(E)); }
template <class W>
__device__ __forceinline__ Extent weight_extent(const NormArgs& a, const void* w) { return Extent(w, (uint64_t)a.C * sizeof(W)); }
__device__ __forceinline__ Extent stats_extent(const NormArgs& a, const float* p) { return Extent(p, (uint64_t)a.rows * a.groups * sizeof(float)); }
template <class E>
__device__ __forceinline__ float get(const E* p, const Extent& in) { return in.holds(p) ? to_f(*p) : 0.f; }
template <class E>
__device__ __forceinline__ void put(E* p, E v, const Extent& out) {
    if (out.holds(p)) *p = v;
}

template <class E, class W>
__global__ void __launch_bounds__(NT) norm_fwd_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[NT / 32];
    const int m = a.C / a.groups;
    for (int64_t unit = blockIdx.x; unit < a.rows * a.groups; unit += gridDim.x) {
    const int64_t row = unit / a.groups;
    const int g = (int)(unit - row * a.groups);
    const E* x = static_cast<const E*>(a.x) + row * a.x_stride + g * m;
    const W *w = static_cast<const W*>(a.w), *b = static_cast<const W*>(a.b);
    const Extent in = x_extent<E>(a);
    float s = 0.f;
    for (int i = threadIdx.x; i < m; i += NT) s += get(x + i, in);
    const float mean = block_sum_nt(s, red) / (float)m;
    float q = 0.f;
    for (int i = threadIdx.x; i < m; i += NT) {
        const float d = get(x + i, in) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(block_sum_nt(q, red) / (float)m + a.eps);
    E* y = static_cast<E*>(a.y) + row * a.C + g * m;
    for (int i = threadIdx.x; i < m; i += NT)
        put(y + i,
            from_f<E>(fmaf((get(x + i, in) - mean) * rstd, w ? get(w + g * m + i, weight_extent<W>(a, w)) : 1.f,
                           b ? get(b + g * m + i, weight_extent<W>(a, b)) : 0.f)),
            dense_extent<E>(a, a.y));
    if (a.mean && threadIdx.x == 0) {
        put(a.mean + unit, mean, stats_extent(a, a.mean));
        put(a.rstd + unit, rstd, stats_extent(a, a.rstd));
    }
    }
}

template <class E, class W>
__global__ void __launch_bounds__(NT) norm_dx_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[NT / 32];
    const int m = a.C / a.groups;
    for (int64_t unit = blockIdx.x; unit < a.rows * a.groups; unit += gridDim.x) {
    const int64_t row = unit / a.groups;
    const int g = (int)(unit - row * a.groups);
    const E *x = static_cast<const E*>(a.x) + row * a.x_stride + g * m, *dy = static_cast<const E*>(a.dy) + row * a.dy_stride + g * m;
    const W* w = static_cast<const W*>(a.w);
    const Extent in = x_extent<E>(a), up = dy_extent<E>(a), weights = weight_extent<W>(a, a.w);
    const float mean = get(a.mean + unit, stats_extent(a, a.mean)), rstd = get(a.rstd + unit, stats_extent(a, a.rstd));
    float s = 0.f, q = 0.f;
    for (int i = threadIdx.x; i < m; i += NT) {
        const float e = get(dy + i, up) * (w ? get(w + g * m + i, weights) : 1.f);
        s += e;
        q = fmaf(e, (get(x + i, in) - mean) * rstd, q);
    }
    s = block_sum_nt(s, red) / (float)m;
    q = block_sum_nt(q, red) / (float)m;
    E* dx = static_cast<E*>(a.dx) + row * a.C + g * m;
    for (int i = threadIdx.x; i < m; i += NT) {
        const float e = get(dy + i, up) * (w ? get(w + g * m + i, weights) : 1.f);
        put(dx + i, from_f<E>(rstd * (e - s - (get(x + i, in) - mean) * rstd * q)), dense_extent<E>(a, a.dx));
    }
    }
}

constexpr int COL_ROWS = 64;   // rows of one block's partial sums

template <class E>
__global__ void __launch_bounds__(NT) norm_cols_kernel(const __grid_constant__ NormArgs a) {
    const int c = blockIdx.x * NT + threadIdx.x, m = a.C / a.groups;
    if (c >= a.C) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float dy = get(static_cast<const E*>(a.dy) + r * a.dy_stride + c, dy_extent<E>(a));
        const int64_t at = r * a.groups + c / m;
        const float x = get(static_cast<const E*>(a.x) + r * a.x_stride + c, x_extent<E>(a));
        db += dy;
        dw = fmaf(dy, (x - get(a.mean + at, stats_extent(a, a.mean))) * get(a.rstd + at, stats_extent(a, a.rstd)), dw);
    }
    put(a.scratch + ((int64_t)blockIdx.y * 2) * a.C + c, dw, Extent(a.scratch, a.scratch_bytes));
    put(a.scratch + ((int64_t)blockIdx.y * 2 + 1) * a.C + c, db, Extent(a.scratch, a.scratch_bytes));
}

// adds up the blocks' sums: 32 columns per block, 16 threads a column, in one order
constexpr int FT = 512;
template <class W>
__global__ void __launch_bounds__(FT) norm_finish_kernel(const __grid_constant__ NormArgs a, int parts) {
    __shared__ float2 red[FT / 32][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    pdl_wait();
    float dw = 0.f, db = 0.f;
    if (c < a.C) {
        const float* p = a.scratch + c;
#pragma unroll 4
        for (int i = g; i < parts; i += FT / 32) {
            dw += get(p + (int64_t)i * 2 * a.C, Extent(a.scratch, a.scratch_bytes));
            db += get(p + ((int64_t)i * 2 + 1) * a.C, Extent(a.scratch, a.scratch_bytes));
        }
    }
    red[g][threadIdx.x & 31] = make_float2(dw, db);
    __syncthreads();
    if (g != 0 || c >= a.C) return;
#pragma unroll
    for (int i = 1; i < FT / 32; ++i) {
        dw += red[i][threadIdx.x].x;
        db += red[i][threadIdx.x].y;
    }
    if (a.dw) put(static_cast<W*>(a.dw) + c, from_f<W>(dw), weight_extent<W>(a, a.dw));
    if (a.db) put(static_cast<W*>(a.db) + c, from_f<W>(db), weight_extent<W>(a, a.db));
}

// ---- rows in pieces of 16 bytes ----------------------------------------------------------------------------------------
// For rows, weights and outputs on 16-byte boundaries; others take the kernels above. A group is a row (its values are spread over a team of TPR
// threads), or SEG lanes of a warp, one piece each.
template <class E>
constexpr int per_piece = 16 / sizeof(E);

template <class E, class W>
__device__ __forceinline__ void load_weights(const W* w, int c, float other, float* f, const Extent& weights) {   // the weights of a piece's columns
    constexpr int N = per_piece<E>;
    if (!w) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = other;
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i += per_piece<W>) {
        const uint4* p = reinterpret_cast<const uint4*>(w + c + i);
        unpack<W>(weights.holds(p) ? __ldg(p) : make_uint4(0, 0, 0, 0), f + i);
    }
}
template <class E, class W>
struct PieceWeights {   // kept as they are stored
    static constexpr int N = per_piece<E>, U = N / per_piece<W>;
    uint4 u[U];
    __device__ __forceinline__ void load(const W* w, int c, const Extent& weights) {
#pragma unroll
        for (int i = 0; i < U; ++i) u[i] = w && weights.holds(reinterpret_cast<const uint4*>(w + c) + i) ? __ldg(reinterpret_cast<const uint4*>(w + c) + i) : ones();
    }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < U; ++i) unpack<W>(u[i], f + i * per_piece<W>);
    }
    static __device__ __forceinline__ uint4 ones() {
        const uint32_t o = sizeof(W) == 4 ? 0x3f800000u : std::is_same<W, __half>::value ? 0x3c003c00u : 0x3f803f80u;
        return make_uint4(o, o, o, o);
    }
};
__device__ __forceinline__ float lanes_sum(float v, int lanes) {   // over aligned runs of `lanes` lanes (a power of two)
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// s / m from 1 / m rounded, by one step on the remainder (which is exact): exact where the quotient is, so that rows of one value have no deviation.
// (The product alone is off by up to 1.5 units, which rows of 1000 whose length is not a power of two showed as 0.019, times 1 / sqrt(eps).)
__device__ __forceinline__ float quotient(float s, float m, float inv_m) {
    const float q = s * inv_m;
    return fmaf(fmaf(-q, m, s), inv_m, q);
}

// One pass over x: a thread keeps NV pieces of its row in registers between the statistics and the output.
// BLOCK: a block per row, else a warp per row; SEG (of a warp's lanes per group): a warp per NV * 32 pieces of a row.
constexpr int BT = 128;   // threads of a row that has a block to itself: a thread's fixed work (addresses, reductions) is shared by 32 or 64 values
template <class E, class W, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? BT : NT) norm_rows_fwd_kernel(const __grid_constant__ NormArgs a, int seg) {
    constexpr int N = per_piece<E>, TPR = BLOCK ? BT : 32;
    __shared__ float red[2][BT / 32];
    const int tid = threadIdx.x, lane = BLOCK ? tid : tid & 31, pieces = a.C / N;
    const int parts = seg ? (pieces + 32 * NV - 1) / (32 * NV) : 1;   // of a row
    const unsigned unit = BLOCK ? blockIdx.x : blockIdx.x * (NT / 32) + (tid >> 5);   // (below 2^32: see fwd_rows)
    const int64_t row = seg ? unit / (unsigned)parts : unit;
    const int p0 = (int)(unit - (unsigned)row * (unsigned)parts) * 32 * NV * (seg ? 1 : 0) + lane;
    if (row >= a.rows) return;
    const E* x = static_cast<const E*>(a.x) + row * a.x_stride;
    const int m = a.C / a.groups;
    const float inv_m = 1.f / (float)m;
    float f[NV][N], mean[NV], rstd[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int p = p0 + j * TPR;
        const uint4* from = reinterpret_cast<const uint4*>(x) + p;
        unpack<E>(p < pieces && x_extent<E>(a).holds(from) ? __ldcs(from) : make_uint4(0, 0, 0, 0), f[j]);
    }
    auto total = [&](float v, float* r) {     // over the row
        v = warp_sum(v);
        if (!BLOCK) return v;
        if ((tid & 31) == 0) r[tid >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < BT / 32; ++i) v += r[i];
        return v;
    };
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float t = 0.f;
#pragma unroll
        for (int c = 0; c < N; ++c) t += f[j][c];
        if (seg) mean[j] = quotient(lanes_sum(t, seg), (float)m, inv_m);
        else s += t;
    }
    if (!seg) {
        s = quotient(total(s, red[0]), (float)m, inv_m);
#pragma unroll
        for (int j = 0; j < NV; ++j) mean[j] = s;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float t = 0.f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            f[j][c] -= mean[j];
            t = fmaf(f[j][c], f[j][c], t);
        }
        if (p0 + j * TPR >= pieces) t = 0.f;
        if (seg) rstd[j] = rsqrtf(lanes_sum(t, seg) * inv_m + a.eps);
        else q += t;
    }
    if (!seg) {
        q = rsqrtf(total(q, red[1]) * inv_m + a.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) rstd[j] = q;
    }
    E* y = static_cast<E*>(a.y) + row * a.C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int p = p0 + j * TPR;
        if (p >= pieces) continue;
        float w[N], b[N];
        load_weights<E>(static_cast<const W*>(a.w), p * N, 1.f, w, weight_extent<W>(a, a.w));
        load_weights<E>(static_cast<const W*>(a.b), p * N, 0.f, b, weight_extent<W>(a, a.b));
#pragma unroll
        for (int c = 0; c < N; ++c) w[c] = fmaf(f[j][c] * rstd[j], w[c], b[c]);
        if (dense_extent<E>(a, a.y).holds(reinterpret_cast<uint4*>(y) + p)) __stcs(reinterpret_cast<uint4*>(y) + p, pack<E>(w));
        if (a.mean && (seg ? p % seg == 0 : p == 0)) {
            const int64_t at = row * a.groups + (seg ? p / seg : 0);
            put(a.mean + at, mean[j], stats_extent(a, a.mean));
            put(a.rstd + at, rstd[j], stats_extent(a, a.rstd));
        }
    }
}

// The backward pass, one read of x and dy: a block per SM, whose copying warp brings rows in ahead (a ring of bulk copies) and whose teams of TPR
// threads take them in turn. A thread keeps the sums of its columns for dw and db from row to row; teams are added up in shared memory at the end,
// blocks by norm_finish_kernel, always in one order.
// (256 threads with twice the values each: 17 % fewer instructions, 71 us instead of 56 at 8192 x 4096 bf16. 96 registers a thread: bf16 rows keep
// within them, fp16 rows of two pieces spill 116 bytes, 72 us, 160 with fp32 weights, and groups 104 to 132.)
constexpr int BWD_THREADS = 512, BWD_RING = 196608;
struct NormBwd {
    NormArgs a;
    int tpr, seg, slots, row_bytes;   // threads per row, lanes per group (0: the row is one), rows in the ring
};
template <class E, class W, int NV, bool SEG>
__global__ void __launch_bounds__(BWD_THREADS + 32, 1) norm_rows_bwd_kernel(const __grid_constant__ NormBwd k) {
    constexpr int N = per_piece<E>, MAX_SLOTS = 64;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ uint64_t full[MAX_SLOTS], vacant[MAX_SLOTS];
    __shared__ float2 red[2][BWD_THREADS / 32];
    __shared__ int failed;
    __shared__ uint32_t nobody;
    const NormArgs& a = k.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, pieces = a.C / N;
    const int tpr = k.tpr, teams = BWD_THREADS / tpr, wpt = tpr / 32;   // warps per team
    if (tid == 0) {
        for (int i = 0; i < k.slots; ++i) mbar_init(&full[i], 1), mbar_init(&vacant[i], wpt);
        fence_mbar_init();
        failed = 0;
    }
    __syncthreads();
    pdl_launch_dependents();
    // after the first wait that runs out nobody waits any more
    auto wait_for = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile int*>(&failed)) return false;
        if (mbar_wait_bounded(bar, parity, 1u << 18)) return true;
        *reinterpret_cast<volatile int*>(&failed) = 1;
        atomicOr(&g_device_status, DEV_WAIT_HEAD);
        return false;
    };
    const int mine = (int)((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);   // rows blockIdx.x, + gridDim.x, ... (no more blocks than rows)
    // a slot of the ring and the phase of its barriers, `by` rows further on
    auto advance = [&](int& slot, uint32_t& phase, int by) {
        slot += by;
        if (slot >= k.slots) slot -= k.slots, phase ^= 1u;
    };
    float dw[NV][N], db[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int c = 0; c < N; ++c) dw[j][c] = db[j][c] = 0.f;
    if (warp == BWD_THREADS / 32) {
        if (lane == 0) {
            int n = 0, slot = 0;
            uint32_t phase = 0;
            for (; n < mine; ++n, advance(slot, phase, 1)) {
                if (n >= k.slots && !wait_for(&vacant[slot], phase ^ 1u)) break;
                const int64_t r = blockIdx.x + (int64_t)n * gridDim.x;
                unsigned char* to = ring + (size_t)slot * 2 * k.row_bytes;
                const E *x = static_cast<const E*>(a.x) + r * a.x_stride, *dy = static_cast<const E*>(a.dy) + r * a.dy_stride;
                if (x_extent<E>(a).holds(x, k.row_bytes / sizeof(E)) && dy_extent<E>(a).holds(dy, k.row_bytes / sizeof(E)) &&
                    AB_BC(slot >= 0 && slot < MAX_SLOTS && (slot + 1) * 2 * k.row_bytes <= BWD_RING)) {
                    mbar_expect_tx(&full[slot], 2 * k.row_bytes);
                    bulk_g2s(to, x, k.row_bytes, &full[slot]);
                    bulk_g2s(to + k.row_bytes, dy, k.row_bytes, &full[slot]);
                } else {
                    mbar_arrive(&full[slot]);
                }
            }
            // whatever became of the waits, all that was asked for lands before the ring is used otherwise, or the block ends
            for (int c = max(0, n - k.slots); c < n; ++c) mbar_wait_bounded(&full[c % k.slots], (uint32_t)(c / k.slots) & 1u, 1u << 18);
        }
    } else {
        const int team = warp / wpt, t = tid - team * tpr;
        const float inv_m = 1.f / (float)(a.C / a.groups);
        PieceWeights<E, W> w[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (t + j * tpr < pieces) w[j].load(static_cast<const W*>(a.w), (t + j * tpr) * N, weight_extent<W>(a, a.w));
        constexpr int NS = SEG ? NV : 1;                  // groups that a thread's pieces belong to
        int group[NS];
        float mean[NS], rstd[NS], mean1[NS], rstd1[NS];   // of a row, and of the team's next one
#pragma unroll
        for (int j = 0; j < NS; ++j) group[j] = SEG ? min(t + j * tpr, pieces - 1) / k.seg : 0;
        auto stats = [&](int n) {
            if (n >= mine) return;
            const int64_t at = (blockIdx.x + (int64_t)n * gridDim.x) * a.groups;
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (stats_extent(a, a.mean).holds(a.mean + at + group[j])) mean1[j] = __ldg(a.mean + at + group[j]), rstd1[j] = __ldg(a.rstd + at + group[j]);
        };
        stats(team);
        int slot = team, turn = 0;
        uint32_t phase = 0;
        for (int n = team; n < mine; n += teams, advance(slot, phase, teams), turn ^= 1) {
            const int64_t r = blockIdx.x + (int64_t)n * gridDim.x;
#pragma unroll
            for (int j = 0; j < NS; ++j) mean[j] = mean1[j], rstd[j] = rstd1[j];
            stats(n + teams);
            wait_for(&full[slot], phase);
            __syncwarp();
            const uint4* from = reinterpret_cast<const uint4*>(ring + (size_t)slot * 2 * k.row_bytes);
            uint4 ux[NV], ud[NV];
            uint32_t used = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int p = t + j * tpr;
                ux[j] = ud[j] = make_uint4(0, 0, 0, 0);
                if (p < pieces) {
                    ux[j] = from[p];
                    ud[j] = from[k.row_bytes / 16 + p];
                }
                used ^= ux[j].x ^ ud[j].x;
            }
            loads_returned(used, &nobody);
            __syncwarp();
            if (lane == 0) mbar_arrive(&vacant[slot]);
            // xh and dy w are worked out again for dx where a row is one group: kept over the block's exchange of sums they cost spills (65 us
            // instead of 56 at 8192 x 4096 bf16; over a few lanes' exchange 30.5 instead of 35.5 at 4097 x 2560 fp16 in groups of 64)
            float s = 0.f, q = 0.f, sj[NS], qj[NS], xh[SEG ? NV : 1][N], e[SEG ? NV : 1][N];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int g = SEG ? j : 0;
                float sp = 0.f, qp = 0.f;
                unpack<E>(ux[j], xh[g]);
                unpack<E>(ud[j], e[g]);
                if (t + j * tpr < pieces) {
                    float fw[N];
                    w[j].get(fw);
#pragma unroll
                    for (int c = 0; c < N; ++c) {
                        xh[g][c] = (xh[g][c] - mean[g]) * rstd[g];
                        dw[j][c] = fmaf(e[g][c], xh[g][c], dw[j][c]);
                        db[j][c] += e[g][c];
                        e[g][c] *= fw[c];
                        sp += e[g][c];
                        qp = fmaf(e[g][c], xh[g][c], qp);
                    }
                }
                if (SEG) {
                    sj[g] = lanes_sum(sp, k.seg) * inv_m;
                    qj[g] = lanes_sum(qp, k.seg) * inv_m;
                } else {
                    s += sp;
                    q += qp;
                }
            }
            if (!SEG) {
                s = warp_sum(s);
                q = warp_sum(q);
                if (wpt > 1) {
                    float2* to = red[turn];   // (written again two rows on, behind the next row's barrier)
                    if (lane == 0) to[warp] = make_float2(s, q);
                    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(tpr) : "memory");
                    s = q = 0.f;
                    for (int i = 0; i < wpt; ++i) {
                        const float2 v = to[team * wpt + i];
                        s += v.x;
                        q += v.y;
                    }
                }
                sj[0] = s * inv_m, qj[0] = q * inv_m;
            }
            if (a.dx) {
                uint4* dx = reinterpret_cast<uint4*>(static_cast<E*>(a.dx) + r * a.C);
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int p = t + j * tpr;
                    if (p >= pieces) continue;
                    const int g = SEG ? j : 0;
                    float fx[N];
                    if (!SEG) {
                        float fw[N];
                        unpack<E>(ux[j], xh[0]);
                        unpack<E>(ud[j], e[0]);
                        w[j].get(fw);
#pragma unroll
                        for (int c = 0; c < N; ++c) xh[0][c] = (xh[0][c] - mean[0]) * rstd[0], e[0][c] *= fw[c];
                    }
#pragma unroll
                    for (int c = 0; c < N; ++c) fx[c] = rstd[g] * fmaf(-xh[g][c], qj[g], e[g][c] - sj[g]);
                    if (dense_extent<E>(a, a.dx).holds(dx + p)) __stcs(dx + p, pack<E>(fx));
                }
            }
        }
    }
    if (!a.dw && !a.db) return;
    // the ring is free: the teams' sums, added up in their order
    float* sums = reinterpret_cast<float*>(ring);   // [teams][C]
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        if (warp < BWD_THREADS / 32) {
            const int team = warp / wpt, t = tid - team * tpr;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (t + j * tpr < pieces)
#pragma unroll
                    for (int c = 0; c < N; ++c)
                        put(sums + team * a.C + (t + j * tpr) * N + c, which ? db[j][c] : dw[j][c], Extent(ring, BWD_RING));
        }
        __syncthreads();
        for (int c = tid; c < a.C; c += BWD_THREADS + 32) {
            float s = 0.f;
            for (int i = 0; i < teams; ++i) s += sums[i * a.C + c];
            put(a.scratch + ((int64_t)blockIdx.x * 2 + which) * a.C + c, s, Extent(a.scratch, a.scratch_bytes));
        }
    }
}

// calls f with a value of the element type, and one of the weights' type
template <class F>
int with_types(int dtype, int wtype, F f) {
    if (dtype == AB_DT_F32) return f(0.f, 0.f);
    if (dtype == AB_DT_F16) return wtype == AB_DT_F32 ? f(__half(), 0.f) : f(__half(), __half());
    return wtype == AB_DT_F32 ? f(__nv_bfloat16(), 0.f) : f(__nv_bfloat16(), __nv_bfloat16());
}

bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How the kernels for pieces take a call; nv 0: they do not.
struct NormShape {
    int nv, tpr, seg;
};
template <class E>
NormShape norm_shape(const NormArgs& a) {
    constexpr int N = per_piece<E>;
    NormShape s = {};
    if (a.C % N || (a.rows > 1 && (a.x_stride % N || a.dy_stride % N)) || !on_16(a.x) || !on_16(a.w) || !on_16(a.b) || !on_16(a.y) || !on_16(a.dy) || !on_16(a.dx)) return s;
    const int pieces = a.C / N;
    if (a.groups > 1) {
        const int lanes = a.C / a.groups / N;
        if ((a.C / a.groups) % N || lanes > 32 || (lanes & (lanes - 1)) || pieces % lanes) return s;
        s.seg = lanes;
    }
    // threads for a row: as few as hold it with two pieces each (the sums of more columns do not fit a thread's registers beside the row)
    s.tpr = 32;
    while (s.tpr < BWD_THREADS && pieces > s.tpr * 2) s.tpr *= 2;
    s.nv = pieces <= s.tpr ? 1 : pieces <= s.tpr * 2 ? 2 : 0;
    return s;
}

template <class E, class W>
int fwd_rows(const NormArgs& a, const NormShape& s, cudaStream_t st, bool* done) {
    constexpr int N = per_piece<E>;
    const int pieces = a.C / N;
    *done = true;
    if (s.seg || pieces <= 32 * 8) {   // a warp per row, or per 64 pieces of groups
        const int nv = s.seg ? (pieces <= 32 ? 1 : 2) : pieces <= 32 ? 1 : pieces <= 64 ? 2 : pieces <= 128 ? 4 : 8;
        const int64_t units = a.rows * (s.seg ? (pieces + 32 * nv - 1) / (32 * nv) : 1), blocks = (units + NT / 32 - 1) / (NT / 32);
        if (units > UINT32_MAX - NT) {
            *done = false;
            return OK;
        }
        auto k = nv == 1 ? norm_rows_fwd_kernel<E, W, 1, false> : nv == 2 ? norm_rows_fwd_kernel<E, W, 2, false> : nv == 4 ? norm_rows_fwd_kernel<E, W, 4, false> : norm_rows_fwd_kernel<E, W, 8, false>;
        k<<<(unsigned)blocks, NT, 0, st>>>(a, s.seg);
    } else if (pieces <= BT * 8 && a.rows <= INT32_MAX) {
        auto k = pieces <= BT * 4 ? norm_rows_fwd_kernel<E, W, 4, true> : norm_rows_fwd_kernel<E, W, 8, true>;
        k<<<(unsigned)a.rows, BT, 0, st>>>(a, 0);
    } else {
        *done = false;
    }
    return check_cuda(cudaGetLastError(), "ab_layer_norm_fwd");
}

template <class W>
int finish(const NormArgs& a, int parts, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.C + 31) / 32);
    cfg.blockDim = dim3(FT);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = parts ? 1 : 0;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, norm_finish_kernel<W>, a, parts), "ab_layer_norm_bwd");
}

template <class E, class W>
int bwd_rows(const NormArgs& a, const NormShape& s, cudaStream_t st) {
    NormBwd k = {a, s.tpr, s.seg, 0, a.C * (int)sizeof(E)};
    k.slots = std::min(64, BWD_RING / (2 * k.row_bytes));
    auto kernel = s.seg ? (s.nv == 1 ? norm_rows_bwd_kernel<E, W, 1, true> : norm_rows_bwd_kernel<E, W, 2, true>)
                        : (s.nv == 1 ? norm_rows_bwd_kernel<E, W, 1, false> : norm_rows_bwd_kernel<E, W, 2, false>);
    static PerDeviceOnce once;
    const DeviceProps* props = nullptr;
    const int st_ = once.run(&props, [&](const DeviceProps&) -> int {
        for (auto f : {norm_rows_bwd_kernel<E, W, 1, true>, norm_rows_bwd_kernel<E, W, 2, true>, norm_rows_bwd_kernel<E, W, 1, false>, norm_rows_bwd_kernel<E, W, 2, false>})
            AB_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, BWD_RING));
        return OK;
    });
    if (st_ != OK) return st_;
    const int blocks = (int)std::min<int64_t>(a.rows, props->n_sm);
    kernel<<<blocks, BWD_THREADS + 32, BWD_RING, st>>>(k);
    const int e = check_cuda(cudaGetLastError(), "ab_layer_norm_bwd");
    return e != OK || (!a.dw && !a.db) ? e : finish<W>(a, blocks, st);
}

// rows of one block's partial sums in norm_cols_kernel, so that the blocks do not outgrow the grid
int64_t col_parts(int64_t rows) { return std::min<int64_t>((rows + COL_ROWS - 1) / COL_ROWS, 32768); }

}  // namespace

size_t layer_norm_scratch_bytes(int64_t rows, int C) {
    // a block's sums in either kernel: at most 256 blocks (SMs), or one per COL_ROWS rows
    return (size_t)std::max<int64_t>(col_parts(rows), std::min<int64_t>(rows, 256)) * 2 * C * sizeof(float);
}

int layer_norm_fwd(const NormArgs& a, cudaStream_t st) {
    return with_types(a.dtype, a.wtype, [&](auto e, auto w) -> int {
        using E = decltype(e);
        using W = decltype(w);
        const NormShape s = norm_shape<E>(a);
        if (s.nv || (a.groups == 1 && s.tpr)) {
            bool done = false;
            const int c = fwd_rows<E, W>(a, s, st, &done);
            if (c != OK || done) return c;
        }
        const int64_t groups = a.rows * a.groups;
        norm_fwd_kernel<E, W><<<(unsigned)std::min<int64_t>(groups, 1 << 20), NT, 0, st>>>(a);
        return check_cuda(cudaGetLastError(), "ab_layer_norm_fwd");
    });
}

int layer_norm_bwd(const NormArgs& a, cudaStream_t st) {
    return with_types(a.dtype, a.wtype, [&](auto e, auto w) -> int {
        using E = decltype(e);
        using W = decltype(w);
        if (a.rows && a.rows <= INT32_MAX && norm_shape<E>(a).nv && current_sm_count() <= 256) return bwd_rows<E, W>(a, norm_shape<E>(a), st);
        if (a.dx && a.rows) norm_dx_kernel<E, W><<<(unsigned)std::min<int64_t>(a.rows * a.groups, 1 << 20), NT, 0, st>>>(a);
        if (a.dw || a.db) {
            const int parts = (int)col_parts(a.rows);
            if (parts) norm_cols_kernel<E><<<dim3((a.C + NT - 1) / NT, parts), NT, 0, st>>>(a);
            const int c = check_cuda(cudaGetLastError(), "ab_layer_norm_bwd");
            return c != OK ? c : finish<W>(a, parts, st);
        }
        return check_cuda(cudaGetLastError(), "ab_layer_norm_bwd");
    });
}

}  // namespace ab
