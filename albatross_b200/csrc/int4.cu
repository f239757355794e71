// Products of a few rows with 4-bit weights in groups:   y[m, n] = sum_k x[m, k] (q[n, k] - z[n, k / G]) s[n, k / G]
//
// What bounds it: reading the codes, half a byte each, and their scales. A warp takes 16 outputs (rows of the matrix) and 128 inputs at a time, a chunk:
// a lane loads 16 bytes of two rows, 32 consecutive codes of each, straight into registers, four chunks ahead (64 KB per SM in flight), and turns
// them into exact fp16 or bf16 by setting them into the last places of a constant and taking that and the zero point away, one operation for two codes
// each. What a lane holds is its own share of the inner indices of eight MMAs (m16n8k16); x lies in shared memory in the order in which the
// codes fall out of their words, 16 bytes for each word.
// An MMA adds up over four lanes, which hold 128 inputs, and those may be of one, two or four groups. Scales are applied to its 32-bit sums, so the groups
// must not meet in it: of its eight columns, a batch row takes as many as there are groups in a chunk, and in each of them only the lanes
// of that group have inputs, the others zeros. For one batch row (where seven columns would be idle) this costs nothing.
//
// Blocks divide the outputs evenly, to single ones (a tile's rows beyond a block's are not loaded); `kw` warps of a block share a tile's inputs and add their sums in one order. Where
// the activations do not fit into shared memory, a cluster of `ks` blocks divides the inputs.
#include <cuda_bf16.h>

#include "train.cuh"

namespace ab {

namespace {

constexpr int I4_WARPS = 16, I4_THREADS = 32 * I4_WARPS;
__host__ __device__ constexpr int i4_ahead(int groups, int nt) { return nt * groups < 8 ? 4 : 3; }   // chunks in flight per warp (as registers allow)
constexpr int I4_X_BYTES = 128 * 1024;       // activations of a block at most
constexpr int I4_BLOCK_TILES = 32;           // tiles of a cluster at most

struct I4Args {
    const uint8_t *w, *zero;   // zero: null, or a byte per group
    const void *scale, *x;
    void* y;
    int64_t x_stride;
    int32_t N, K, rows;
    int32_t groups;            // of a row
    int32_t per_group;         // chunks of a group (groups of 128 and more; else 1)
    int32_t pass;              // batch rows of a block
    int32_t clusters, ks, kw;
    int32_t x_bytes;           // shared memory: activations, then the warps' sums, then (ks > 1) the block's
};

template <class E> struct I4Type;
template <> struct I4Type<__half> {
    // two codes each: 0 and 4, 1 and 5, 2 and 6, 3 and 7 of a word
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&a)[4]) {
        a[0] = (w & 0x000f000fu) | 0x64006400u;   // 1024 + q
        a[1] = (w & 0x00f000f0u) | 0x54005400u;   // 64 + q
        w >>= 8;
        a[2] = (w & 0x000f000fu) | 0x64006400u;
        a[3] = (w & 0x00f000f0u) | 0x54005400u;
    }
    static __device__ __forceinline__ void less(uint32_t (&a)[4], uint32_t z) {   // z: the zero point in both halves
        const uint32_t even = z | 0x64006400u, odd = (z << 4) | 0x54005400u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = i & 1 ? odd : even;
            const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&a[i]), *reinterpret_cast<const __half2*>(&t));
            a[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ void first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct I4Type<__nv_bfloat16> {
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&a)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;   // 128 + q
    }
    static __device__ __forceinline__ void less(uint32_t (&a)[4], uint32_t z) {
        const uint32_t t = z | 0x43004300u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a[i]), *reinterpret_cast<const __nv_bfloat162*>(&t));
            a[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ void first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ uint4 i4_load(const uint4* p) {
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// where `on` is false the registers keep what they have, with no instruction for it
__device__ __forceinline__ void i4_x(uint4& v, const uint4* p, bool on) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n @p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "r"(smem_u32(p)), "r"((uint32_t)on) : "memory");
}
__device__ __forceinline__ float i4_peer(const float* own, uint32_t rank) {
    float v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}" : "=f"(v) : "r"(smem_u32(own)), "r"(rank) : "memory");
    return v;
}

// GROUPS: of a chunk (1: groups of 128 or more, 2: of 64, 4: of 32). NT: eights of MMA columns, each 8 / GROUPS batch rows.
template <class E, int GROUPS, int NT>
__global__ void __launch_bounds__(I4_THREADS, 1) int4_rows_kernel(const __grid_constant__ I4Args a) {
    extern __shared__ __align__(16) unsigned char i4_smem[];
    using T = I4Type<E>;
    constexpr int AHEAD = i4_ahead(GROUPS, NT);
    constexpr int MR = NT * 8 / GROUPS, SCALES = GROUPS == 1 ? 1 : 2;   // batch rows; scales of a lane's two columns
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int cl = (int)blockIdx.x / a.ks, rank = (int)blockIdx.x - cl * a.ks;
    const int n0 = (int)((int64_t)a.N * cl / a.clusters), n1 = (int)((int64_t)a.N * (cl + 1) / a.clusters), tiles = (n1 - n0 + 15) / 16;
    const int m0 = blockIdx.y * a.pass, rows = min(a.pass, a.rows - m0);
    const int all_chunks = (a.K + 127) / 128;
    const int c0 = (int)((int64_t)all_chunks * rank / a.ks), nc = (int)((int64_t)all_chunks * (rank + 1) / a.ks) - c0;   // of this block
    const int kw = a.kw, slot = warp / kw, kwi = warp - slot * kw, slots = I4_WARPS / kw;
    const int lo = nc * kwi / kw, len = nc * (kwi + 1) / kw - lo;                                                     // of this warp
    const int rounds = slot < tiles ? (tiles - slot + slots - 1) / slots : 0, total = rounds * len;
    uint4* sx = reinterpret_cast<uint4*>(i4_smem);
    float* sums = reinterpret_cast<float*>(i4_smem + a.x_bytes);
    float* block_sums = sums + I4_WARPS * 16 * MR;
    const Extent w_all(a.w, (uint64_t)a.N * (a.K / 2)), s_all(a.scale, (uint64_t)a.N * a.groups * sizeof(E)), z_all(a.zero, (uint64_t)a.N * a.groups);
    pdl_wait();

    // What a chunk needs, in a ring of registers. Addresses are made once for a tile; a chunk is 64 bytes further than the one before.
    uint4 w[AHEAD][2];
    E s[AHEAD][2][SCALES];
    uint32_t z[AHEAD][2];
    int in_tile = slot, in_c = 0;
    bool on[2];
    uint32_t w_at[2], s_at[2];   // in 16 bytes; in groups (32 bits hold them: checked by the launch)
    const int first = c0 + lo, of_code = GROUPS == 1 ? 0 : t * GROUPS / 4;   // the group, of a chunk, of this lane's codes
    // where a row ends inside of a chunk: chunks of this warp in which this lane has codes, and (from its columns) scales
    const int codes_to = GROUPS == 1 ? INT32_MAX : (a.K - t * 32 + 127) / 128 - first;
    auto open = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = n0 + in_tile * 16 + h * 8 + g;
            on[h] = n < n1;
            const uint32_t row = on[h] ? n : n0;
            w_at[h] = row * (uint32_t)(a.K / 32) + first * 4 + t;
            s_at[h] = row * (uint32_t)a.groups + (GROUPS > 1 || a.per_group == 1 ? first * GROUPS : 0);
        }
    };
    auto request = [&](uint4 (&w)[2], E (&s)[2][SCALES], uint32_t (&z)[2]) {
        const int group = GROUPS > 1 || a.per_group == 1 ? in_c * GROUPS : (first + in_c) / a.per_group;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4* p_w = reinterpret_cast<const uint4*>(a.w) + (w_at[h] + in_c * 4);
            w[h] = make_uint4(0, 0, 0, 0);
            if (on[h] && in_c < codes_to && w_all.holds(p_w)) w[h] = i4_load(p_w);
#pragma unroll
            for (int i = 0; i < SCALES; ++i) {
                const int at = group + (SCALES == 1 ? 0 : (2 * t + i) % GROUPS);
                const E* p = static_cast<const E*>(a.scale) + (s_at[h] + at);
                s[h][i] = from_f<E>(0.f);
                if (on[h] && (GROUPS == 1 || first * GROUPS + at < a.groups) && s_all.holds(p)) s[h][i] = __ldg(p);
            }
            z[h] = 8;
            const uint8_t* p_z = a.zero + (s_at[h] + group + of_code);
            if (a.zero && on[h] && in_c < codes_to && z_all.holds(p_z)) z[h] = __ldg(p_z);
        }
        if (++in_c == len) {
            in_c = 0, in_tile += slots;
            open();
        }
    };
    open();
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (i < total) request(w[i], s[i], z[i]);

    // Activations: 16 bytes for each word of codes, [chunk][word of a lane][batch row][lane's quarter].
    {
        const E* x = static_cast<const E*>(a.x) + (int64_t)m0 * a.x_stride;
        const Extent x_all = rows_extent(a.x, a.rows, a.x_stride, a.K, sizeof(E));
        const bool wide = ((reinterpret_cast<uintptr_t>(x) | (uint64_t)a.x_stride * sizeof(E)) & 15) == 0;
        for (int i = threadIdx.x; i < nc * 16 * rows; i += I4_THREADS) {
            const int m = i / (nc * 16), piece = i - m * (nc * 16), c = piece >> 4, quarter = (piece >> 2) & 3, word = piece & 3;
            const int k = (c0 * 16 + piece) * 8;
            const E* p = x + (int64_t)m * a.x_stride + k;
            uint32_t v[4] = {0, 0, 0, 0};
            if (k < a.K && x_all.holds(p, 8)) {
                if (wide) {
                    const uint4 q = *reinterpret_cast<const uint4*>(p);
                    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
                } else {
                    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
                }
            }
            sx[(c * 4 + word) * (rows * 4) + m * 4 + quarter] =
                make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632), __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
        }
    }
    __syncthreads();

    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
    // Where this lane's inputs lie: of its column's batch row, if they are of its column's group; else its registers stay zero. (Columns behind the last batch
    // row read that one's, and nobody reads them.)
    const bool has = GROUPS == 1 || of_code == g % GROUPS;
    const uint4* x_at[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x_at[n] = sx + min(n * (8 / GROUPS) + g / GROUPS, rows - 1) * 4 + t;
    uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};   // (in turn)
    auto chunk = [&](const uint4 (&w)[2], const E (&s)[2][SCALES], const uint32_t (&z)[2], int c) {
        float d[NT][4];
        const uint32_t zl = z[0] * 0x00010001u, zh = z[1] * 0x00010001u;
#pragma unroll
        for (int word = 0; word < 4; ++word) {
            uint32_t l[4], h[4];
            T::codes(word == 0 ? w[0].x : word == 1 ? w[0].y : word == 2 ? w[0].z : w[0].w, l);
            T::codes(word == 0 ? w[1].x : word == 1 ? w[1].y : word == 2 ? w[1].z : w[1].w, h);
            T::less(l, zl);
            T::less(h, zh);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint4& v = x[(word * NT + n) & 1];
                i4_x(v, x_at[n] + (c * 4 + word) * (rows * 4), has && AB_BC((c * 4 + word + 1) * rows * 64 <= a.x_bytes));
                if (word == 0) T::first(d[n], l[0], h[0], l[1], h[1], v.x, v.y);
                else T::mma(d[n], l[0], h[0], l[1], h[1], v.x, v.y);
                T::mma(d[n], l[2], h[2], l[3], h[3], v.z, v.w);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[n][e] = fmaf(to_f(s[e >> 1][SCALES == 1 ? 0 : e & 1]), d[n][e], sum[n][e]);
    };
    auto store = [&](int n, int m, float v) {
        E* y = static_cast<E*>(a.y) + (int64_t)(m0 + m) * a.N + n;
        if (AB_BC(n >= 0 && n < a.N && m >= 0 && m0 + m < a.rows)) *y = from_f<E>(v);
    };
    // the tile's sums: [warp][batch row][output]
    auto finish = [&](int tile) {
        auto meet = [&]() {
            if (kw == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(kw * 32) : "memory");
        };
        meet();   // the tile before has been read
        float* own = sums + warp * (16 * MR);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (GROUPS == 1) {
                    own[(n * 8 + 2 * t) * 16 + g + 8 * h] = sum[n][2 * h];
                    own[(n * 8 + 2 * t + 1) * 16 + g + 8 * h] = sum[n][2 * h + 1];
                } else {
                    float v = sum[n][2 * h] + sum[n][2 * h + 1];
                    if (GROUPS == 4) v += __shfl_xor_sync(0xffffffffu, v, 1);
                    if (GROUPS == 2 || (t & 1) == 0) own[(n * (8 / GROUPS) + 2 * t / GROUPS) * 16 + g + 8 * h] = v;
                }
                sum[n][2 * h] = sum[n][2 * h + 1] = 0.f;
            }
        }
        meet();
        const float* first = sums + slot * kw * (16 * MR);
        for (int e = kwi * 32 + lane; e < 16 * rows; e += kw * 32) {
            float v = 0.f;
            for (int i = 0; i < kw; ++i) v += first[i * (16 * MR) + e];
            const int n = n0 + tile * 16 + (e & 15), m = e >> 4;
            if (a.ks > 1) block_sums[tile * (16 * MR) + e] = v;
            else if (n < n1) store(n, m, v);
        }
    };
    int tile = slot, c = 0;
    if (len == 0)   // (fewer chunks than warps of a tile: this one adds zeros)
        for (int i = 0; i < rounds; ++i) finish(slot + i * slots);
    for (int i = 0; i < total; i += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (i + j < total) {
                chunk(w[j], s[j], z[j], lo + c);
                if (i + j + AHEAD < total) request(w[j], s[j], z[j]);
                if (++c == len) {
                    finish(tile);
                    c = 0, tile += slots;
                }
            }
        }
    }
    if (a.ks > 1) {   // the blocks of a cluster finish its tiles in turn
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = rank; i < tiles; i += a.ks)
            for (int e = threadIdx.x; e < 16 * rows; e += I4_THREADS) {
                float v = 0.f;
                for (int r = 0; r < a.ks; ++r) v += i4_peer(block_sums + i * (16 * MR) + e, (uint32_t)r);
                const int n = n0 + i * 16 + (e & 15);
                if (n < n1) store(n, e >> 4, v);
            }
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <class E, int GROUPS, int NT>
int i4_launch(I4Args a, cudaStream_t st) {
    constexpr int MR = NT * 8 / GROUPS, MOST = I4_X_BYTES + (I4_WARPS + I4_BLOCK_TILES) * 16 * MR * 4;
    static_assert(MOST <= 227 * 1024, "shared memory of the 4-bit products");
    static PerDeviceOnce once;
    const DeviceProps* dev;
    const auto kernel = int4_rows_kernel<E, GROUPS, NT>;
    const int err = once.run(&dev, [&](const DeviceProps& d) -> int {
        AB_CHECK_ARG(d.smem_optin >= (size_t)MOST, "linear_int4: %zu bytes of shared memory per block are too few", d.smem_optin);
        return check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST), "cudaFuncSetAttribute(linear_int4)");
    });
    if (err != OK) return err;
    AB_CHECK_ARG((int64_t)a.N * (a.K / 32) < UINT32_MAX, "linear_int4: a matrix of %d x %d is too large", a.N, a.K);
    const int chunks = (a.K + 127) / 128;
    a.pass = MR < a.rows ? MR : a.rows;
    a.ks = 1;
    while ((int64_t)((chunks + a.ks - 1) / a.ks) * 256 * a.pass > I4_X_BYTES) {
        if (a.ks < 8) a.ks *= 2;
        else if (a.pass > 1) a.pass = (a.pass + 1) / 2;
        else AB_CHECK_ARG(false, "linear_int4: %d inputs are too many", a.K);
    }
    const int nc = (chunks + a.ks - 1) / a.ks;
    a.x_bytes = nc * 256 * a.pass;
    const int fit = dev->n_sm / a.ks;
    a.clusters = a.N < fit ? a.N : fit;
    if (a.ks > 1 && (a.N + a.clusters - 1) / a.clusters > 16 * I4_BLOCK_TILES) a.clusters = (a.N + 16 * I4_BLOCK_TILES - 1) / (16 * I4_BLOCK_TILES);
    // warps that share a tile: the fewest rounds of chunks, a tile's end counted as two of them
    const int tiles = ((a.N + a.clusters - 1) / a.clusters + 15) / 16;
    int best = 0;
    for (int kw = I4_WARPS; kw >= 1; kw /= 2) {
        const int slots = I4_WARPS / kw, cost = (tiles + slots - 1) / slots * ((nc + kw - 1) / kw + 2);
        if (best == 0 || cost < best) best = cost, a.kw = kw;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.clusters * a.ks, (a.rows + a.pass - 1) / a.pass);
    cfg.blockDim = dim3(I4_THREADS);
    cfg.dynamicSmemBytes = a.x_bytes + (I4_WARPS + (a.ks > 1 ? tiles : 0)) * 16 * MR * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.ks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.ks > 1 ? 2 : 1;
    AB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    return OK;
}
template <class E, int GROUPS>
int i4_columns(const I4Args& a, cudaStream_t st) {
    const int tiles = (a.rows * GROUPS + 7) / 8;
    // (16 batch rows are two eights in groups of 128, and four in groups of 64; four in groups of 32 are 8 rows)
    if (tiles <= 1) return i4_launch<E, GROUPS, 1>(a, st);
    if constexpr (GROUPS > 1) {
        if (tiles > 2) return i4_launch<E, GROUPS, 4>(a, st);
    }
    return i4_launch<E, GROUPS, 2>(a, st);
}
template <class E>
int i4_groups(const I4Args& a, int group, cudaStream_t st) {
    return group == 32 ? i4_columns<E, 4>(a, st) : group == 64 ? i4_columns<E, 2>(a, st) : i4_columns<E, 1>(a, st);
}

}  // namespace

int linear_int4(const ab_int4& m, int rows, const void* x, int64_t x_stride, void* y, cudaStream_t st) {
    I4Args a = {};
    a.w = static_cast<const uint8_t*>(m.w), a.zero = static_cast<const uint8_t*>(m.zero), a.scale = m.scale, a.x = x, a.y = y, a.x_stride = x_stride;
    a.N = m.n_out, a.K = m.k, a.rows = rows, a.groups = m.k / m.group, a.per_group = m.group > 128 ? m.group / 128 : 1;
    return m.dtype == AB_DT_F16 ? i4_groups<__half>(a, m.group, st) : i4_groups<__nv_bfloat16>(a, m.group, st);
}

}  // namespace ab
