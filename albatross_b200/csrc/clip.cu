// The norm over many tensors of gradients, and clipping.
//
//   norm = scale sqrt(sum of g^2 over all tensors),   out = f g,   f = scale min(1, max_norm / norm)   (scale alone where the norm is not
//                                                     finite in 32 bits)
//
// What bounds it: memory. The factor depends on every value, so that the gradients are read twice, and the floor (each read once) is out of reach
// for what does not stay in L2.
//
// Two launches whatever the number of tensors: the list travels as a kernel parameter (up to 32 KB), which a captured graph keeps a copy
// of. All tensors make one row of units, 16 bytes of a tensor each; what is in front of a tensor's first 16-byte boundary and behind its
// last one is one more unit. Warps take 256 units at a time, across the ends of tensors, so that small vectors between large matrices cost
// no more than their bytes. The first launch leaves one sum per block; each block of the second adds them all up in the same order (so the
// factor is the same everywhere, and the result does not depend on the order in which blocks run), and goes through the units backwards:
// what was read last is still in L2.
//
// Precision: eight squares are added up in 32 bits, what comes of that in 64 (a unit's sum is 2e-7 off at most, the norm of many units
// 1e-8). Where 32 bits could overflow or lose small squares (bf16 and fp32), the unit is done again in 64. An output is rounded to 32 bits
// and then to its type; the first of the two can move the second by 2^-24 of the value, which is below a 2^-13th of a 16-bit step.
//
// Measured: the squares of 0.38 GB of fp16 60 us (6.4 TB/s), the scaling into fp32 190 (0.38 read, 0.76 written: 6.1 TB/s; some of it comes
// from L2 where calls follow one another). In place, 2.7 GB of bf16: 1.30 ms, 6.3 TB/s for the three passes. A list of little tensors costs
// the host 0.04 to 0.1 us each in place and 0.07 to 0.2 into others, beside some 11; the GPU 13 to 16 us in place for 20 to 440 tensors of
// 100 values and 20 to 33 into others, one after the other by the warps that have them.
#include <type_traits>

#include "train.cuh"

namespace ab {

namespace {

constexpr int CL_THREADS = 512, CL_WARPS = CL_THREADS / 32;
constexpr int CL_LOADS = 8;                     // units in flight per lane
constexpr uint32_t CL_SHARE = 32 * CL_LOADS;    // units that a warp takes at a time
constexpr int CL_BLOCKS_PER_SM = 2;
// The list of a launch: few tensors in a small parameter (a launch copies all of it), many in the largest there is: 20 tensors 12 us of the
// host's time, and 20 in the large one; 65 tensors 16 and 23, 110 tensors 19 and 25.
constexpr int CL_FEW = 120, CL_MANY = 1000;

struct ClipTensor {
    const void* g;
    void* out;
    uint64_t n;
    uint32_t first;        // first unit
    uint16_t head;         // values in front of the first 16-byte boundary
    uint8_t types;         // type of g, and of out in bits 2 and 3
    uint8_t out_apart;     // how a unit's outputs lie: 0 on a boundary of their size, 1 on one of 16 bytes (they have 32), 2 elsewhere: stored value by value
};
template <int CAP>
struct ClipList {
    uint32_t units;        // of all tensors
    int32_t n;
    ClipTensor t[CAP];
};
static_assert(sizeof(ClipList<CL_MANY>) + 64 <= 32764, "parameters of the clipping kernels");

__host__ __device__ constexpr int clip_per_unit(int type) { return type == AB_DT_F32 ? 4 : 8; }

// the tensor that unit u belongs to
template <int CAP>
__device__ __forceinline__ int clip_find(const ClipList<CAP>& list, uint32_t u) {
    int lo = 0, hi = list.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.t[mid].first <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double clip_block_sum(double v, double* s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[threadIdx.x & (CL_WARPS - 1)];
#pragma unroll
    for (int o = CL_WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;   // every thread has it
}

template <class E>
__device__ __forceinline__ double unit_squares(const uint4& q) {
    constexpr int N = 16 / sizeof(E);
    float f[N];
    unpack<E>(q, f);
    float s = f[0] * f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) s = fmaf(f[i], f[i], s);
    if (sizeof(E) == 2 && std::is_same<E, __half>::value) return s;   // 2^-48 .. 2^35: 32 bits hold it
    if (s > 1e-25f && s < 1e37f) return s;
    constexpr uint32_t M = sizeof(E) == 2 ? 0x7fff7fffu : 0x7fffffffu;
    if (((q.x | q.y | q.z | q.w) & M) == 0) return 0.0;               // (gradients of rows that nobody looked at)
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fma((double)f[i], (double)f[i], d);
    return d;
}

template <class E>
__device__ __forceinline__ uint32_t clip_whole(const ClipTensor& t) { return (uint32_t)((t.n - t.head) / (16 / sizeof(E))); }

template <class E>
__device__ __forceinline__ double squares_of(const ClipTensor& t, uint32_t lo, uint32_t hi, int lane) {   // units lo .. hi - 1 of the tensor
    const Extent all(t.g, t.n * sizeof(E));
    const E* g = static_cast<const E*>(t.g);
    const uint4* body = reinterpret_cast<const uint4*>(g + t.head);
    const uint32_t whole = clip_whole<E>(t), end = min(hi, whole);
    double sum = 0.0;
    uint4 q[CL_LOADS];
#pragma unroll
    for (int i = 0; i < CL_LOADS; ++i) {
        const uint32_t u = lo + i * 32 + lane;
        q[i] = u < end && all.holds(body + u) ? __ldg(body + u) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < CL_LOADS; ++i) sum += unit_squares<E>(q[i]);
    if (hi > whole) {   // the unit of the edges
        const uint64_t behind = t.head + (uint64_t)whole * (16 / sizeof(E));
        const uint64_t at = lane < t.head ? lane : behind + (lane - t.head);
        if (at < t.n && all.holds(g + at)) {
            const double v = to_f(g[at]);
            sum = fma(v, v, sum);
        }
    }
    return sum;
}

template <int CAP>
__global__ void __launch_bounds__(CL_THREADS, CL_BLOCKS_PER_SM) grad_squares_kernel(const __grid_constant__ ClipList<CAP> list, double* __restrict__ sums) {
    __shared__ double s[CL_WARPS];
    const int lane = threadIdx.x & 31;
    pdl_launch_dependents();
    double sum = 0.0;
    // (64 bits: the share behind the last one may begin beyond 2^32)
    for (uint64_t at = ((uint64_t)blockIdx.x * CL_WARPS + (threadIdx.x >> 5)) * CL_SHARE; at < list.units; at += (uint64_t)gridDim.x * CL_WARPS * CL_SHARE) {
        const uint32_t end = (uint32_t)min((uint64_t)list.units, at + CL_SHARE);
        uint32_t u = (uint32_t)at;
        for (int i = clip_find(list, u); u < end; ++i) {
            const ClipTensor& t = list.t[i];
            const uint32_t stop = i + 1 < list.n ? min(end, list.t[i + 1].first) : end;
            const int type = t.types & 3;
            if (type == AB_DT_F16) sum += squares_of<__half>(t, u - t.first, stop - t.first, lane);
            else if (type == AB_DT_BF16) sum += squares_of<__nv_bfloat16>(t, u - t.first, stop - t.first, lane);
            else sum += squares_of<float>(t, u - t.first, stop - t.first, lane);
            u = stop;
        }
    }
    sum = clip_block_sum(sum, s);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// 32 bytes at once: as two stores of 16, each lane's halves lie 32 bytes apart, and the two cost as much as whole lines each
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}

// The factor, as 32 bits and a power of two: a norm of up to 2^128 leaves a limit's quotient below 2^-126, where 32 bits have few places.
// (A scale is below 2^128.)
struct ClipFactor {
    float f;
    bool small;
    __device__ __forceinline__ explicit ClipFactor(double v) : f((float)(v < 0x1p-126 ? v * 0x1p126 : v)), small(v < 0x1p-126) {}
    __device__ __forceinline__ float of(float v) const { return small ? v * f * 0x1p-126f : v * f; }
};

template <class E, class O>
__device__ __forceinline__ void scale_units(const ClipTensor& t, uint32_t lo, uint32_t hi, ClipFactor f, int lane) {
    constexpr int N = 16 / sizeof(E), W = N * sizeof(O) / 16;   // stores of 16 bytes per unit (0: of 8)
    const Extent all(t.g, t.n * sizeof(E)), all_out(t.out, t.n * sizeof(O));
    const E* g = static_cast<const E*>(t.g);
    O* out = static_cast<O*>(t.out);
    const uint4* body = reinterpret_cast<const uint4*>(g + t.head);
    const uint32_t whole = clip_whole<E>(t), end = min(hi, whole);
    uint4 q[CL_LOADS];
#pragma unroll
    for (int i = 0; i < CL_LOADS; ++i) {
        const uint32_t u = lo + i * 32 + lane;
        q[i] = u < end && all.holds(body + u) ? __ldcs(body + u) : make_uint4(0, 0, 0, 0);   // (not __ldg: out may be g)
    }
#pragma unroll
    for (int i = 0; i < CL_LOADS; ++i) {
        const uint32_t u = lo + i * 32 + lane;
        if (u >= end) continue;
        float v[N];
        unpack<E>(q[i], v);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = f.of(v[k]);
        O* to = out + t.head + (uint64_t)u * N;
        if (!all_out.holds(to, N)) continue;
        if (t.out_apart == 2) {
#pragma unroll
            for (int k = 0; k < N; ++k) to[k] = from_f<O>(v[k]);
        } else if (W == 2 && t.out_apart == 0) {
            store32(to, pack<O>(v), pack<O>(v + 16 / sizeof(O) % N));
        } else if (W == 0) {
            O half_[8];
#pragma unroll
            for (int k = 0; k < N; ++k) half_[k] = from_f<O>(v[k]);
            __stcs(reinterpret_cast<uint2*>(to), *reinterpret_cast<const uint2*>(half_));
        } else {
#pragma unroll
            for (int k = 0; k < W; ++k) __stcs(reinterpret_cast<uint4*>(to) + k, pack<O>(v + k * (16 / sizeof(O))));
        }
    }
    if (hi > whole) {
        const uint64_t behind = t.head + (uint64_t)whole * N;
        const uint64_t at = lane < t.head ? lane : behind + (lane - t.head);
        if (at < t.n && all.holds(g + at) && all_out.holds(out + at)) out[at] = from_f<O>(f.of(to_f(g[at])));
    }
}
template <class E>
__device__ __forceinline__ void scale_units_to(int type, const ClipTensor& t, uint32_t lo, uint32_t hi, ClipFactor f, int lane) {
    if (type == AB_DT_F16) scale_units<E, __half>(t, lo, hi, f, lane);
    else if (type == AB_DT_BF16) scale_units<E, __nv_bfloat16>(t, lo, hi, f, lane);
    else scale_units<E, float>(t, lo, hi, f, lane);
}

struct ClipHow {
    const double* sums;
    int32_t n_sums;
    int32_t in_place;      // every out is its g, and of its type: nothing is to be done where the factor is 1
    int32_t writes;        // 0: the norm alone is wanted
    double scale, max_norm;
    float* norm;           // null: another launch of the same call writes it
};

template <int CAP>
__global__ void __launch_bounds__(CL_THREADS, CL_BLOCKS_PER_SM) grad_scale_kernel(const __grid_constant__ ClipList<CAP> list, const __grid_constant__ ClipHow how) {
    __shared__ double s[CL_WARPS];
    const int lane = threadIdx.x & 31;
    pdl_wait();
    double sum = 0.0;
    for (int i = threadIdx.x; i < how.n_sums; i += CL_THREADS) sum += how.sums[i];
    sum = clip_block_sum(sum, s);
    const double norm = how.scale * sqrt(sum);
    if (how.norm && blockIdx.x == 0 && threadIdx.x == 0) *how.norm = (float)norm;
    // (not finite: as it is handed out. A norm beyond 32 bits is an infinity to the caller, who is told that nothing is clipped then)
    const ClipFactor f(norm > how.max_norm && (float)norm < INFINITY ? how.scale * (how.max_norm / norm) : how.scale);
    if (!how.writes || (how.in_place && f.f == 1.f && !f.small)) return;
    const uint64_t shares = ((uint64_t)list.units + CL_SHARE - 1) / CL_SHARE;
    for (uint64_t i = (uint64_t)blockIdx.x * CL_WARPS + (threadIdx.x >> 5); i < shares; i += (uint64_t)gridDim.x * CL_WARPS) {
        const uint64_t at = (shares - 1 - i) * CL_SHARE;
        const uint32_t end = (uint32_t)min((uint64_t)list.units, at + CL_SHARE);
        uint32_t u = (uint32_t)at;
        for (int k = clip_find(list, u); u < end; ++k) {
            const ClipTensor& t = list.t[k];
            const uint32_t stop = k + 1 < list.n ? min(end, list.t[k + 1].first) : end;
            const int type = t.types & 3, to = t.types >> 2;
            if (type == AB_DT_F16) scale_units_to<__half>(to, t, u - t.first, stop - t.first, f, lane);
            else if (type == AB_DT_BF16) scale_units_to<__nv_bfloat16>(to, t, u - t.first, stop - t.first, f, lane);
            else scale_units_to<float>(to, t, u - t.first, stop - t.first, f, lane);
            u = stop;
        }
    }
}

// up to CAP tensors from t[from] on
template <int CAP>
int clip_list(const ab_grad* t, int64_t from, int64_t n, ClipList<CAP>& list) {
    list.n = 0;
    uint64_t units = 0;
    for (int64_t i = from; i < n && i < from + CAP; ++i) {
        const int size = t[i].dtype == AB_DT_F32 ? 4 : 2, out_size = t[i].out_dtype == AB_DT_F32 ? 4 : 2, per = clip_per_unit(t[i].dtype);
        if (t[i].n == 0) continue;
        ClipTensor& e = list.t[list.n];
        e.g = t[i].g, e.out = t[i].out, e.n = (uint64_t)t[i].n, e.first = (uint32_t)units;
        const uint64_t head = (16 - (reinterpret_cast<uintptr_t>(e.g) & 15)) % 16 / size;
        e.head = (uint16_t)(head < e.n ? head : e.n);
        e.types = (uint8_t)(t[i].dtype | t[i].out_dtype << 2);
        // a unit's outputs: 8 bytes (32 bits into 16), 16 or 32
        const uint64_t bytes = per * out_size, to = reinterpret_cast<uintptr_t>(e.out) + (uint64_t)e.head * out_size;
        e.out_apart = to % bytes == 0 ? 0 : bytes == 32 && to % 16 == 0 ? 1 : 2;
        units += (e.n - e.head) / per + (e.head != 0 || (e.n - e.head) % per != 0 ? 1 : 0);
        AB_CHECK_ARG(units < UINT32_MAX, "clip_grad_norm: the tensors of a launch have too many values");
        ++list.n;
    }
    list.units = (uint32_t)units;
    return OK;
}

template <int CAP>
int clip_launch(const ab_grad* t, int64_t n, bool writes, double scale, double max_norm, float* norm, double* sums, cudaStream_t st) {
    const int most = current_sm_count() * CL_BLOCKS_PER_SM;
    ClipList<CAP> list;
    auto blocks = [&]() {
        const uint64_t wanted = ((uint64_t)list.units + CL_SHARE * CL_WARPS - 1) / (CL_SHARE * CL_WARPS);
        return (int)(wanted < 1 ? 1 : wanted > (uint64_t)most ? most : wanted);
    };
    ClipHow how = {sums, 0, 1, writes ? 1 : 0, scale, max_norm, norm};
    for (int64_t from = 0; from == 0 || from < n; from += CAP) {   // the squares of all lists
        const int err = clip_list(t, from, n, list);
        if (err != OK) return err;
        for (int i = 0; i < list.n; ++i)
            if (list.t[i].g != list.t[i].out || (list.t[i].types & 3) != list.t[i].types >> 2) how.in_place = 0;
        const int grid = blocks();
        grad_squares_kernel<CAP><<<grid, CL_THREADS, 0, st>>>(list, sums + how.n_sums);
        AB_CUDA(cudaGetLastError());
        how.n_sums += grid;
    }
    for (int64_t from = 0; from == 0 || (writes && from < n); from += CAP) {   // then the scaling
        if (n > CAP) {
            const int err = clip_list(t, from, n, list);
            if (err != OK) return err;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(writes ? blocks() : 1);
        cfg.blockDim = dim3(CL_THREADS);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = from == 0 ? 1 : 0;   // (it begins while the last sums are made; further launches follow one another)
        AB_CUDA(cudaLaunchKernelEx(&cfg, grad_scale_kernel<CAP>, list, how));
        how.norm = nullptr;
    }
    return OK;
}

}  // namespace

size_t clip_scratch_bytes(int64_t n) { return (size_t)((n + CL_MANY - 1) / CL_MANY + 1) * current_sm_count() * CL_BLOCKS_PER_SM * sizeof(double); }

int clip_grad_norm(const ab_grad* t, int64_t n, bool writes, double scale, double max_norm, float* norm, double* sums, cudaStream_t st) {
    return n <= CL_FEW ? clip_launch<CL_FEW>(t, n, writes, scale, max_norm, norm, sums, st) : clip_launch<CL_MANY>(t, n, writes, scale, max_norm, norm, sums, st);
}

}  // namespace ab
