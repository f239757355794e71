// Products of a few rows with 4-bit weights in groups:   y[m, n] = sum_k x[m, k] (q[n, k] - z[n, k / G]) s[n, k / G]
//
// What bounds it: reading the codes, half a byte each, and their scales. Every warp streams pieces of its own, 32 outputs (rows of the
// matrix) by 256 inputs, into a ring in shared memory (TMA, 4 KB, 128 to 192 KB per SM in flight); nobody else is waited for until a tile
// of 32 outputs is done. It turns codes into exact fp16 or bf16 by setting them into the last places of a constant and taking that and the
// zero point away, one operation each for two codes. A lane's 16 bytes of a row, 32 codes, are its own share of the inner indices of eight
// MMAs (m16n8k16); x lies in shared memory in the order in which codes fall out of their words, 16 bytes for each word.
// An MMA adds up over four lanes, which hold 128 inputs, and those may be of one, two or four groups. Scales are applied to its 32-bit
// sums, so the groups must not meet in it: of its eight columns, a batch row takes as many as there are groups in 128 inputs, and in each
// of them only the lanes of that group have inputs, the others zeros. For one batch row (where seven columns would be idle) this costs
// nothing.
//
// Blocks divide the outputs evenly, to single ones (the tiles of a block are as high as its share asks for), and a block's warps its
// pieces, tile after tile: a warp stores the tiles that it has to itself, leaves its sums of those that it shares in shared memory, and at
// the end they are added up in one order. Nobody waits before that. Where the activations do not fit into shared memory, or the outputs are
// few, a cluster of `ks` blocks divides the inputs.
//
// Measured, one batch row: 65536 x 4096 fp16 in groups of 128 33 us, 4.2 TB/s of codes and scales (27 with the arithmetic left out: 5.1);
// 4096 x 4096 7.4 (6.3), of which some 6 are the launch, the activations and the way to the first piece. Beyond the streaming, no unit is
// near its rate: the warps issue 147 instructions for 2048 codes, 2.2 a cycle and SM of 4, the ALU pipe is 45 % busy and the matrix unit 24
// %, with 16 warps an SM (a quarter of what it holds): what is left is waiting, for a piece's words, for each other's results and for the
// scales, which come by loads of 4 bytes from eight rows. More warps or fewer (24, 8), codes taken as subnormal numbers (132 instructions)
// and zero points taken out by sums of the inputs were no faster, the last two slower in groups of 32 and with eight rows (20.5 -> 26).
// More rows than one pass takes cost a pass each, whatever their number: 16 rows of 65536 x 4096 81 us, 64 of 16384 x 4096 in groups of 64
// 184, 320 of them 989, 2048 of 4096 x 4096 642.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "gemm.cuh"
#include "train.cuh"

namespace ab {

namespace {

constexpr int I4_WARPS = 16, I4_THREADS = 32 * I4_WARPS;
constexpr int I4_ROWS = 32, I4_PIECE = I4_ROWS * 128;   // a piece: 128 bytes of up to 32 rows
constexpr int I4_STAGES = 3;                 // pieces in flight per warp (two where shared memory is needed elsewhere)
constexpr int I4_SMEM = 225 * 1024;
constexpr int I4_SHARED = 2 * I4_WARPS;      // sums of shared tiles: a warp's first and its last

struct I4Args {
    const uint8_t* zero;       // null, or a byte per group
    const void *scale, *x;
    void* y;
    int64_t x_stride;
    int32_t N, K, rows;
    int32_t groups;            // of a row
    int32_t per_group;         // chunks (of 128 inputs) of a group (groups of 128 and more; else 1)
    int32_t pairs;             // two scales next to each other are 4 bytes on their boundary
    int32_t pass;              // batch rows of a block
    int32_t clusters, ks, height, stages;
    int32_t x_bytes;           // shared memory: the rings, then activations, the warps' sums, and (ks > 1) those of the block's tiles
};

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {   // one operation (as operators, two immediates made two of it)
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(a), "r"(mask), "r"(bits));
    return v;
}
template <class E> struct I4Type;
template <> struct I4Type<__half> {
    // two codes each: 0 and 4, 1 and 5, 2 and 6, 3 and 7 of a word
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&a)[4]) {
        a[0] = and_or(w, 0x000f000fu, 0x64006400u);   // 1024 + q
        a[1] = and_or(w, 0x00f000f0u, 0x54005400u);   // 64 + q
        w >>= 8;
        a[2] = and_or(w, 0x000f000fu, 0x64006400u);
        a[3] = and_or(w, 0x00f000f0u, 0x54005400u);
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
        for (int i = 0; i < 4; ++i) a[i] = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);   // 128 + q
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

__device__ __forceinline__ void i4_tma(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y),
                 "r"(smem_u32(bar)) : "memory");
}
// where `on` is false the registers keep what they have, with no instruction for it
__device__ __forceinline__ void i4_x(uint4& v, uint32_t p, uint32_t on) {
    asm("{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n @p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n}" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "r"(p), "r"(on));
}
__device__ __forceinline__ float i4_peer(const float* own, uint32_t rank) {
    float v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}" : "=f"(v) : "r"(smem_u32(own)), "r"(rank) : "memory");
    return v;
}

// GROUPS: of a chunk (1: groups of 128 or more, 2: of 64, 4: of 32). NT: eights of MMA columns, each 8 / GROUPS batch rows.
template <class E, int GROUPS, int NT, bool ZERO>
__global__ void __launch_bounds__(I4_THREADS, 1) int4_rows_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ I4Args a) {
    extern __shared__ __align__(1024) unsigned char i4_smem[];
    __shared__ uint64_t full[I4_WARPS][I4_STAGES];
    __shared__ int first_tile[I4_WARPS];
    __shared__ uint32_t s_nobody;
    using T = I4Type<E>;
    constexpr int PAIRS = GROUPS == 1 ? 1 : 2;     // pairs of scales of a lane and row: of the piece's two chunks, or in each of them of its two columns
    constexpr int MS = NT <= 2 ? 2 : 1;            // halves of a tile that share what is read of the activations (as registers allow)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int cl = (int)blockIdx.x / a.ks, rank = (int)blockIdx.x - cl * a.ks;
    const int n0 = (int)((int64_t)a.N * cl / a.clusters), n1 = (int)((int64_t)a.N * (cl + 1) / a.clusters), tiles = (n1 - n0 + a.height - 1) / a.height;
    const int m0 = blockIdx.y * a.pass, rows = min(a.pass, a.rows - m0);
    const int all_pieces = (a.K + 255) / 256;
    const int c0 = (int)((int64_t)all_pieces * rank / a.ks), nc = (int)((int64_t)all_pieces * (rank + 1) / a.ks) - c0;   // of this block
    auto run_of = [&](int w) { return tiles * nc * w / I4_WARPS; };   // pieces through all tiles: a warp's first
    const int run0 = run_of(warp), total = run_of(warp + 1) - run0;
    const int tile0 = run0 / nc, in0 = run0 - tile0 * nc;
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)i4_smem + 1023) & ~(uintptr_t)1023);
    unsigned char* ring = base + warp * a.stages * I4_PIECE;
    uint4* sx = reinterpret_cast<uint4*>(base + I4_WARPS * a.stages * I4_PIECE);
    float* sums = reinterpret_cast<float*>(base + I4_WARPS * a.stages * I4_PIECE + a.x_bytes);
    float* block_sums = sums + I4_SHARED * I4_ROWS * rows;
    const Extent s_all(a.scale, (uint64_t)a.N * a.groups * sizeof(E)), z_all(a.zero, (uint64_t)a.N * a.groups);
    if (lane == 0) {
        for (int i = 0; i < a.stages; ++i) mbar_init(&full[warp][i], 1);
        fence_mbar_init();
        first_tile[warp] = tile0;
    }
    __syncwarp();
    pdl_launch_dependents();
    if (threadIdx.x == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    pdl_wait();   // (codes and scales too may have been written just before)

    // The warp's pieces one behind the other, tile after tile; its first lane asks for them, a.stages ahead of the one worked on.
    int in_i = 0, in_c = in0, in_row = n0 + tile0 * a.height, in_stage = 0;
    auto request = [&]() {   // (one lane)
        if (in_i >= total) return;
        uint64_t* bar = &full[warp][in_stage];
        mbar_expect_tx(bar, (uint32_t)a.height * 128u);
        i4_tma(ring + in_stage * I4_PIECE, &map, (c0 + in_c) * 128, in_row, bar);
        ++in_i;
        if (++in_stage == a.stages) in_stage = 0;
        if (++in_c == nc) in_c = 0, in_row += a.height;
    };
    if (lane == 0)
        for (int i = 0; i < a.stages; ++i) request();

    // Scales and zero points of a piece, in registers, one piece ahead: of rows g, g + 8, g + 16 and g + 24 of the tile. Rows behind the
    // tile's, whose sums nobody reads, take the last one's, and so do groups behind a row's, whose inputs are zeros.
    struct Scales {
        uint32_t s[4][PAIRS], z[ZERO ? 4 : 1];   // z: of the first chunk, and of the second one in the high half
    };
    const int of_code = GROUPS == 1 ? 0 : t * GROUPS / 4;   // the group, of a chunk, of this lane's codes
    const unsigned short* scale = static_cast<const unsigned short*>(a.scale);
    uint32_t s_row[4];
    auto scale_rows = [&](int tile) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s_row[r] = (uint32_t)min(n0 + tile * a.height + r * 8 + g, n1 - 1) * (uint32_t)a.groups;
    };
    auto load_scales = [&](int c, Scales& v) {
        const int chunk = 2 * (c0 + c), last = a.groups - 1;
        if (a.pairs) {
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                const int group = min(GROUPS == 1 ? chunk : (chunk + p) * GROUPS + 2 * t % GROUPS, last - 1);
#pragma unroll
                for (int r = 0; r < 4; ++r) v.s[r][p] = s_all.holds(scale + s_row[r] + group, 2) ? __ldg(reinterpret_cast<const uint32_t*>(scale + (s_row[r] + group))) : 0u;
            }
        } else {
#pragma unroll 1
            for (int p = 0; p < PAIRS; ++p) {
                const int first = GROUPS == 1 ? chunk / a.per_group : (chunk + p) * GROUPS + 2 * t % GROUPS, second = GROUPS == 1 ? (chunk + 1) / a.per_group : first + 1;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const unsigned short *l = scale + s_row[r] + min(first, last), *h = scale + s_row[r] + min(second, last);
                    const uint32_t two = s_all.holds(l) && s_all.holds(h) ? __ldg(l) | (uint32_t)__ldg(h) << 16 : 0u;
                    if (p == 0) v.s[r][0] = two;
                    else v.s[r][PAIRS - 1] = two;
                }
            }
        }
        if (ZERO) {
            const int l = min(GROUPS == 1 ? (a.per_group == 1 ? chunk : chunk / a.per_group) : chunk * GROUPS + of_code, last);
            const int h = min(GROUPS == 1 ? (a.per_group == 1 ? chunk + 1 : (chunk + 1) / a.per_group) : (chunk + 1) * GROUPS + of_code, last);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint8_t *zl = a.zero + (s_row[r] + l), *zh = a.zero + (s_row[r] + h);
                v.z[r] = z_all.holds(zl) && z_all.holds(zh) ? __ldg(zl) | (uint32_t)__ldg(zh) << 16 : 0u;
            }
        }
    };
    Scales cur, next;
    scale_rows(tile0);
    if (total > 0) load_scales(in0, next);

    // Activations: 16 bytes for each word of codes, [chunk][word of a lane][batch row][lane's quarter]; zeros behind the last input.
    {
        const E* x = static_cast<const E*>(a.x) + (int64_t)m0 * a.x_stride;
        const Extent x_all = rows_extent(a.x, a.rows, a.x_stride, a.K, sizeof(E));
        const bool wide = ((reinterpret_cast<uintptr_t>(x) | (uint64_t)a.x_stride * sizeof(E)) & 15) == 0;
        constexpr int AT_ONCE = 4;   // loads of a thread in flight (one after the other 8 rows of 4096 took 3 us)
        const int eights = nc * 32 * rows;
        for (int i0 = threadIdx.x; i0 < eights; i0 += AT_ONCE * I4_THREADS) {
            uint32_t v[AT_ONCE][4];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int i = i0 + j * I4_THREADS, m = i / (nc * 32), k = (c0 * 32 + i - m * (nc * 32)) * 8;
                const E* p = x + (int64_t)m * a.x_stride + k;
                v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0;
                if (i < eights && k < a.K && x_all.holds(p, 8)) {
                    if (wide) {
                        const uint4 q = *reinterpret_cast<const uint4*>(p);
                        v[j][0] = q.x, v[j][1] = q.y, v[j][2] = q.z, v[j][3] = q.w;
                    } else {
                        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[j][e] = h[2 * e] | (uint32_t)h[2 * e + 1] << 16;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int i = i0 + j * I4_THREADS, m = i / (nc * 32), eight = i - m * (nc * 32), c = eight >> 4, quarter = (eight >> 2) & 3, word = eight & 3;
                if (i < eights)
                    sx[(c * 4 + word) * (rows * 4) + m * 4 + quarter] = make_uint4(__byte_perm(v[j][0], v[j][2], 0x5410), __byte_perm(v[j][0], v[j][2], 0x7632),
                                                                                   __byte_perm(v[j][1], v[j][3], 0x5410), __byte_perm(v[j][1], v[j][3], 0x7632));
            }
        }
    }
    __syncthreads();

    float sum[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) sum[m][n][0] = sum[m][n][1] = sum[m][n][2] = sum[m][n][3] = 0.f;
    // Where this lane's inputs lie: of its column's batch row, if they are of its column's group; else its registers stay zero. (Columns
    // behind the last batch row read that one's, and nobody reads them.)
    const bool has = GROUPS == 1 || of_code == g % GROUPS;
    uint32_t x_at[NT];   // (defined behind the barrier: what reads through them cannot be moved in front of it)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        x_at[n] = smem_u32(sx + min(n * (8 / GROUPS) + g / GROUPS, rows - 1) * 4 + t);
        asm volatile("" : "+r"(x_at[n])::"memory");
    }
    uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};   // (in turn)
    const uint32_t has_it = has, x_word = rows * 64;
    auto low = [](uint32_t v) { return from_bits<E>((unsigned short)v); };
    auto high = [](uint32_t v) { return from_bits<E>((unsigned short)(v >> 16)); };
    // The piece's two chunks. (Not unrolled: the code of both did not fit the instruction cache's first level.) Returns a combination of a
    // word of each load from the stage.
    auto piece = [&](const unsigned char* w, Scales& v, int c) -> uint32_t {
        uint32_t used = 0, x_c = (uint32_t)c * 8 * x_word;
        const unsigned char* w_at = w + g * 128 + ((t ^ g) << 4);   // (the second chunk's 16 bytes: bit 6 of the address)
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch, x_c += 4 * x_word) {
            const unsigned char* w_ch = reinterpret_cast<const unsigned char*>(reinterpret_cast<uintptr_t>(w_at) ^ (uintptr_t)(ch * 64));
#pragma unroll
            for (int mb = 0; mb < 2; mb += MS) {
                float d[MS][NT][4];
                uint4 q[MS][2];
#pragma unroll
                for (int m = 0; m < MS; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        q[m][h] = *reinterpret_cast<const uint4*>(w_ch + (16 * (mb + m) + 8 * h) * 128);
                        used ^= q[m][h].x;
                    }
#pragma unroll
                for (int word = 0; word < 4; ++word) {
                    uint32_t l[MS][4], h[MS][4];
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        T::codes(word == 0 ? q[m][0].x : word == 1 ? q[m][0].y : word == 2 ? q[m][0].z : q[m][0].w, l[m]);
                        T::codes(word == 0 ? q[m][1].x : word == 1 ? q[m][1].y : word == 2 ? q[m][1].z : q[m][1].w, h[m]);
                        T::less(l[m], ZERO ? __byte_perm(v.z[ZERO ? 2 * (mb + m) : 0], 0, 0x1010) : 0x00080008u);
                        T::less(h[m], ZERO ? __byte_perm(v.z[ZERO ? 2 * (mb + m) + 1 : 0], 0, 0x1010) : 0x00080008u);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint4& b = x[(word * NT + n) & 1];
                        i4_x(b, x_at[n] + x_c + word * x_word, has_it && AB_BC(x_c + (word + 1) * x_word <= (uint32_t)a.x_bytes));
#pragma unroll
                        for (int m = 0; m < MS; ++m) {
                            if (word == 0) T::first(d[m][n], l[m][0], h[m][0], l[m][1], h[m][1], b.x, b.y);
                            else T::mma(d[m][n], l[m][0], h[m][0], l[m][1], h[m][1], b.x, b.y);
                            T::mma(d[m][n], l[m][2], h[m][2], l[m][3], h[m][3], b.z, b.w);
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < MS; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t two = v.s[2 * (mb + m) + (e >> 1)][0];
                            sum[mb + m][n][e] = fmaf(to_f(PAIRS == 1 || (e & 1) == 0 ? low(two) : high(two)), d[m][n][e], sum[mb + m][n][e]);
                        }
            }
            // the second chunk's
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v.s[r][0] = PAIRS == 1 ? v.s[r][0] >> 16 : v.s[r][PAIRS - 1];
                if (ZERO) v.z[ZERO ? r : 0] >>= 16;
            }
        }
        return used;
    };
    auto store = [&](int n, int m, float v) {
        E* y = static_cast<E*>(a.y) + (int64_t)(m0 + m) * a.N + n;
        if (AB_BC(n >= 0 && n < a.N && m >= 0 && m0 + m < a.rows)) *y = from_f<E>(v);
    };
    // the sum of an output and batch row goes to its place, or (ks > 1) to the block's sums
    auto put = [&](int tile, int in_tile, int m, float v) {
        const int n = n0 + tile * a.height + in_tile;
        if (in_tile >= a.height || n >= n1) return;
        if (a.ks > 1) block_sums[(tile * rows + m) * I4_ROWS + in_tile] = v;
        else store(n, m, v);
    };
    auto finish = [&](int tile, bool alone, int at) {
        float* own = sums + at * I4_ROWS * rows;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = sum[half][n][e];
                    sum[half][n][e] = 0.f;
                    if (GROUPS > 1) {   // the columns of a batch row: this lane's two, and with four groups the next lane's
                        if (e & 1) continue;
                        v += sum[half][n][e + 1];
                        if (GROUPS == 4) v += __shfl_xor_sync(0xffffffffu, v, 1);
                        if (GROUPS == 4 && (t & 1)) continue;
                    }
                    const int m = GROUPS == 1 ? n * 8 + 2 * t + (e & 1) : n * (8 / GROUPS) + 2 * t / GROUPS, in_tile = half * 16 + g + 8 * (e >> 1);
                    if (m >= rows) continue;
                    if (alone) put(tile, in_tile, m, v);
                    else own[m * I4_ROWS + in_tile] = v;
                }
            }
    };
    bool failed = false;
    int tile = tile0, c = in0, stage = 0;
    uint32_t parity = 0;
    for (int i = 0; i < total; ++i) {
        cur = next;
        const bool last = c + 1 == nc;
        if (i + 1 < total) {
            if (last) scale_rows(tile + 1);
            load_scales(last ? 0 : c + 1, next);
        }
        if (!failed && !mbar_wait_bounded(&full[warp][stage], parity, 1u << 16)) failed = true;
        const uint32_t used = piece(ring + stage * I4_PIECE, cur, c);
        loads_returned(used, &s_nobody);
        __syncwarp();   // every lane has read the stage
        if (lane == 0 && !failed) request();
        if (++stage == a.stages) stage = 0, parity ^= 1u;
        if (last || i + 1 == total) {   // alone: all of the tile's pieces were this warp's
            finish(tile, last && i + 1 >= nc, 2 * warp + (tile != tile0));
            ++tile;
        }
        c = last ? 0 : c + 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tiles * rows * I4_ROWS; i += I4_THREADS) {   // the tiles that warps share
        const int tile = i / (rows * I4_ROWS), e = i - tile * (rows * I4_ROWS);
        // warps w with a part of it: those from the last that begins at its first piece or before, on
        int w = tile * I4_WARPS / tiles;
        while (w > 0 && run_of(w) > tile * nc) --w;
        while (run_of(w + 1) <= tile * nc) ++w;
        if (run_of(w) <= tile * nc && run_of(w + 1) >= (tile + 1) * nc) continue;   // (it has all of it, and has stored it)
        float v = 0.f;
        for (; w < I4_WARPS && run_of(w) < (tile + 1) * nc; ++w)
            if (run_of(w) < run_of(w + 1)) v += sums[(2 * w + (tile != first_tile[w])) * I4_ROWS * rows + e];   // (with fewer pieces than warps some have none)
        put(tile, e % I4_ROWS, e / I4_ROWS, v);
    }
    if (a.ks > 1) {   // the blocks of a cluster finish its tiles in turn
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = rank; i < tiles; i += a.ks)
            for (int e = threadIdx.x; e < I4_ROWS * rows; e += I4_THREADS) {
                const int in_tile = e % I4_ROWS, n = n0 + i * a.height + in_tile;
                if (in_tile >= a.height || n >= n1) continue;
                float v = 0.f;
                for (int r = 0; r < a.ks; ++r) v += i4_peer(block_sums + i * rows * I4_ROWS + e, (uint32_t)r);
                store(n, e / I4_ROWS, v);
            }
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (failed) {   // (copies on their way still find their shared memory)
        if (lane == 0) atomicOr(&g_device_status, DEV_WAIT_GEMM);
        for (int i = 0; i < 100; ++i) __nanosleep(1000);
    }
}

template <class E, int GROUPS, int NT, bool ZERO>
int i4_launch(const void* codes, I4Args a, cudaStream_t st) {
    constexpr int MR = NT * 8 / GROUPS, ROOM = I4_SMEM - 1024 - 2 * I4_WARPS * I4_PIECE;   // beside two stages
    static PerDeviceOnce once;
    static int fits[AB_MAX_DEVICES][4];   // clusters of 1, 2, 4 and 8 blocks that a device holds at a time
    const DeviceProps* dev;
    const auto kernel = int4_rows_kernel<E, GROUPS, NT, ZERO>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    auto configure = [&](int clusters, int ks, int passes, int smem) {
        cfg.gridDim = dim3(clusters * ks, passes);
        cfg.blockDim = dim3(I4_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = ks;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = ks > 1 ? 2 : 1;
    };
    const int err = once.run(&dev, [&](const DeviceProps& d) -> int {
        AB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, I4_SMEM));
        fits[&d - once.props][0] = d.n_sm;
        for (int i = 1; i < 4; ++i) {
            configure(1, 1 << i, 1, I4_SMEM);
            AB_CUDA(cudaOccupancyMaxActiveClusters(&fits[&d - once.props][i], kernel, &cfg));
            AB_CHECK_ARG(fits[&d - once.props][i] > 0, "linear_int4: the device holds no cluster of %d blocks", 1 << i);
        }
        return OK;
    });
    if (err != OK) return err;
    AB_CHECK_ARG((int64_t)a.N * (a.K / 32) < UINT32_MAX, "linear_int4: a matrix of %d x %d is too large", a.N, a.K);
    const int pieces = (a.K + 255) / 256;
    a.pass = MR < a.rows ? MR : a.rows;
    // The blocks of a cluster divide the inputs where activations do not fit otherwise, and where outputs are few: then each loads a share
    // of the activations, and has tiles of 32 outputs instead of single ones, as long as two of them hold its outputs. 1 row, groups of
    // 128, undivided against four and eight blocks: 1024 x 4096 7.4 us, 7.2, 5.9; 512 x 16384 13.1, 8.7, 7.5; 2048 x 8224 (groups of 32)
    // 11.1, 9.6, 10.3; 4096 x 8224 11.9, 13.0, 13.7.
    int tiles = 0, shared = 0, lg = 0;   // of a block; shared memory behind the activations; of ks
    const int* const fit_of = fits[dev - once.props];
    for (const int l : {3, 2})
        if (lg == 0 && pieces >= 1 << l && a.N <= 2 * I4_ROWS * fit_of[l]) lg = l;
    for (a.ks = 1 << lg;;) {
        const int64_t x_bytes = (int64_t)((pieces + a.ks - 1) / a.ks) * 512 * a.pass;
        const int tile_bytes = I4_ROWS * a.pass * 4;
        if (x_bytes + (I4_SHARED + (a.ks > 1 ? 8 : 0)) * tile_bytes <= ROOM) {
            const int passes = (a.rows + a.pass - 1) / a.pass;
            const int most = a.ks > 1 ? (int)((ROOM - x_bytes) / tile_bytes - I4_SHARED) * I4_ROWS : a.N;   // outputs whose sums fit
            // All passes at once, one turn of clusters (their beginning is paid once; 1024 x 4096 in groups of 32, 16 rows 23.7 -> 12.2),
            // unless the sums of so many outputs do not fit.
            int fit = std::max(1, fit_of[lg] / passes);
            if ((a.N + fit - 1) / fit > most) fit = fit_of[lg];
            a.x_bytes = (int)x_bytes;
            a.clusters = a.N < fit ? a.N : fit;
            if ((a.N + a.clusters - 1) / a.clusters > most) a.clusters = (a.N + most - 1) / most;
            if (a.clusters > fit && a.pass > 8) {   // more turns than one: rather two passes of half the rows (16 rows: 4096 x 4096 26.4 -> 11.9, 65536 x 4096 248 -> 80)
                a.pass = (a.pass + 1) / 2, lg = 0, a.ks = 1;
                continue;
            }
            const int share = (a.N + a.clusters - 1) / a.clusters;
            tiles = (share + I4_ROWS - 1) / I4_ROWS;
            a.height = (share + tiles - 1) / tiles;
            shared = (I4_SHARED + (a.ks > 1 ? tiles : 0)) * tile_bytes;
            break;
        }
        if (a.ks < 8) a.ks *= 2, ++lg;
        else if (a.pass > 1) a.pass = (a.pass + 1) / 2;
        else AB_CHECK_ARG(false, "linear_int4: %d inputs are too many", a.K);
    }
    AB_CHECK_ARG((int64_t)tiles * ((pieces + a.ks - 1) / a.ks) * I4_WARPS <= INT32_MAX, "linear_int4: a matrix of %d x %d is too large", a.N, a.K);
    a.stages = std::min(I4_STAGES, (I4_SMEM - 1024 - a.x_bytes - shared) / (I4_WARPS * I4_PIECE));
    a.pairs = a.per_group == 1 && a.groups % 2 == 0 && (reinterpret_cast<uintptr_t>(a.scale) & 3) == 0;
    EncodeTiledFn encode;
    const int found = get_encode_fn(&encode);
    if (found != OK) return found;
    CUtensorMap map;
    const cuuint64_t dim[2] = {(cuuint64_t)a.K / 2, (cuuint64_t)a.N}, pitch[1] = {(cuuint64_t)a.K / 2};
    const cuuint32_t box[2] = {128, (cuuint32_t)a.height}, step[2] = {1, 1};
    const CUresult cr = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dim, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) {
        set_error("linear_int4: cuTensorMapEncodeTiled failed with %d (%d x %d)", (int)cr, a.N, a.K);
        return ERR_CUDA;
    }
    configure(a.clusters, a.ks, (a.rows + a.pass - 1) / a.pass, 1024 + a.stages * I4_WARPS * I4_PIECE + a.x_bytes + shared);
    AB_CUDA(cudaLaunchKernelEx(&cfg, kernel, map, a));
    return OK;
}
template <class E, int GROUPS, int NT>
int i4_zeros(const void* codes, const I4Args& a, cudaStream_t st) {
    return a.zero ? i4_launch<E, GROUPS, NT, true>(codes, a, st) : i4_launch<E, GROUPS, NT, false>(codes, a, st);
}
template <class E, int GROUPS>
int i4_columns(const void* codes, const I4Args& a, cudaStream_t st) {
    const int tiles = (a.rows * GROUPS + 7) / 8;
    // (16 batch rows are two eights in groups of 128, and four in groups of 64; four in groups of 32 are 8 rows)
    if (tiles <= 1) return i4_zeros<E, GROUPS, 1>(codes, a, st);
    if constexpr (GROUPS > 1) {
        if (tiles > 2) return i4_zeros<E, GROUPS, 4>(codes, a, st);
    }
    return i4_zeros<E, GROUPS, 2>(codes, a, st);
}
template <class E>
int i4_groups(const void* codes, const I4Args& a, int group, cudaStream_t st) {
    return group == 32 ? i4_columns<E, 4>(codes, a, st) : group == 64 ? i4_columns<E, 2>(codes, a, st) : i4_columns<E, 1>(codes, a, st);
}

}  // namespace

int linear_int4(const ab_int4& m, int rows, const void* x, int64_t x_stride, void* y, cudaStream_t st) {
    I4Args a = {};
    a.zero = static_cast<const uint8_t*>(m.zero), a.scale = m.scale, a.x = x, a.y = y, a.x_stride = x_stride;
    a.N = m.n_out, a.K = m.k, a.rows = rows, a.groups = m.k / m.group, a.per_group = m.group > 128 ? m.group / 128 : 1;
    return m.dtype == AB_DT_F16 ? i4_groups<__half>(m.w, a, m.group, st) : i4_groups<__nv_bfloat16>(m.w, a, m.group, st);
}

}  // namespace ab
