// One id per row of logits, drawn under a temperature, top-k, top-p and min-p from a given uniform number.
//
//   w_i = exp((l_i - max l) / T);  the values in order: larger ones first, equals by index.  Kept is the longest front part of that order in which
//   each value but the first has   rank < k,   sum of the w in front of it < p * (sum of w over the first k),   w >= m.
//   The id is the first one whose sum of w up to and with it exceeds u * (sum of w that is kept).
//
// All three filters keep a front part of one and the same order, and so does the draw: each is a question "where in that order do the
// weights (or the ranks) reach X?". What bounds it is less the reading of a row (it stays in shared memory, of one block or of a cluster's)
// than what is done for each of its values, so the way goes by what the filters leave:
//   few values    top-k up to 600 over the row's blocks, or min-p: the k-th largest of the threads' own maxima is a bound that some k
//                 values and a few more reach. Those are gathered, sorted, and their weights added up: every question is answered among
//                 them, without an exponential for any other value.
//   a bracket     else the sum over the row is needed: 32-bit exponentials and a histogram of counts over 4096 bins of max - l in one
//                 pass. A bin's counts bound its weights within a percent, so they say in which few bins X is reached; their values are
//                 gathered and sorted, and what lies in front of them is added up in 32 bits (nothing, where the values down to there are
//                 few). Those sums are off by EPS at most: where that might move a border across the place, or the bracket holds more than
//                 1024 values, it is done again in whole numbers.
//   whole numbers a histogram over the same bins with exact sums, by atomics on shared memory; its running sums answer every question down
//                 to a bin. The few values of that bin are gathered and compared with each other; where they are more than SP_LIST (ties
//                 of 16-bit logits), the bin's keys' range is divided again.
//
// Precision: weights are taken as multiples of 2^-44 (the largest is 2^44 of them), so that sums are whole numbers and do not depend on the
// order of additions; they come from a table and a polynomial in 64 bits (off by 1e-15). What comes out is the id that the definition in 64
// bits gives, unless u or p meets a border within some 1e-9 of the sum. The log-probability has the 32-bit sum where a bracket sufficed:
// off by EPS.
//
// Measured, fp32 x 65536: one row under top-p 0.9 19 to 27 us, 44 to 60 where it comes to whole numbers (a third of the rows of normal
// logits with a deviation of 1, a sixth with 2, a thirtieth with 3; under top-p 0.99 most), 11 under min-p 0.05, 42 where that keeps more
// than 1024 values; 512 rows under top-p 0.9 317, without filters 223, two blocks a row, of which an SM holds one. What bounds them: the
// shared memory that a row takes (92 KB beside up to 129 of the row: one block an SM), and three or four passes over it, one with an atomic
// for each value. 16-bit rows of up to 65536 values and a small top-k of the same k have kernels of their own, below.
#include <cooperative_groups.h>

#include "train.cuh"

namespace ab {

namespace {

namespace cg = cooperative_groups;

constexpr int SP_BINS = 4096, SP_SUB = 1024;   // bins of the first histogram, and of a division of one of its bins
constexpr int SP_LIST = 256;                   // values that are compared with each other
constexpr int SP_MAX_BLOCKS = 8;               // of a cluster: a row's at most
constexpr int SP_ROW_BYTES = 129 * 1024;       // of a row in a block's shared memory, at most
constexpr uint64_t SP_ONE = 1ull << 44;        // a weight of 1

struct SampleArgs {
    const void* logits;
    const float *u, *T, *p, *m;   // T, p, m: null, or one per row
    const int32_t* k;
    double T_all, p_all, m_all;
    int32_t k_all, V;
    int64_t rows, stride;
    int64_t* ids;
    float* logp;
    int32_t share;                // 16-byte pieces of a row that a block takes
    int32_t ahead;                // rows from one that is worked on to the one that follows it there
};

__device__ __forceinline__ uint32_t key_of(float v) {   // larger values, larger keys; -0 is 0
    const uint32_t b = __float_as_uint(v + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

struct RowScale {
    float top;          // the row's largest value
    float bins;         // bins per unit of top - l
    double c;           // log2(e) / T
    const double* tab;  // 2^(j / 16), j = 0 .. 15
};
__device__ __forceinline__ int bin_of(const RowScale& r, float v) {   // never falls as v does; rounding and all
    const float d = v == r.top ? 0.f : r.top - v;
    return (int)(__float_as_uint(fminf(d * r.bins, SP_BINS - 1) + 8388608.f) & (2 * SP_BINS - 1));   // (2^23: the last places are whole numbers. A conversion has a quarter of the rate)
}
// w in 32 bits, by the hardware's 2^x (relative error 2^-22). The product's rounding and what 32 bits leave of c are made good, so that
// 2^-22 + 2^-23 remains, and 2^-24 z ln 2 for the rounding of the difference d: below 2^-20 for z up to 22 (values beyond that weigh 2^-4
// of the largest at most, all together). 16-bit logits are no better there: 513 and a number of 2^-15 are 26 bits apart. d is finite.
__device__ __forceinline__ float weight32(float d, float c, float c_low) {
    const float z = d * c, rest = fmaf(d, c_low, fmaf(d, c, -z));
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(-z));
    return fmaf(w * -0.693147181f, rest, w);
}
// exp((v - top) / T): 2^z with z = n / 16 + f, |f| <= 1 / 32, and the series of exp(f ln 2) to the sixth power (what is left is below 5e-16)
__device__ __forceinline__ double weight(const RowScale& r, float v) {
    if (v == r.top) return 1.0;
    const double z = ((double)v - (double)r.top) * r.c;
    if (!(z > -46.0)) return 0.0;
    constexpr double ROUND = 6755399441055744.0;   // 1.5 * 2^52
    const double b = fma(z, 16.0, ROUND);
    const int n = (int)(uint32_t)__double_as_longlong(b);
    const double x = fma(b - ROUND, -0.0625, z) * 0.693147180559945309417;
    double q = fma(x, 1.0 / 720.0, 1.0 / 120.0);
    q = fma(q, x, 1.0 / 24.0);
    q = fma(q, x, 1.0 / 6.0);
    q = fma(q, x, 0.5);
    q = fma(q, x, 1.0);
    q = fma(q, x, 1.0) * r.tab[n & 15];
    return __longlong_as_double(__double_as_longlong(q) + ((long long)(n >> 4) << 52));
}
__device__ __forceinline__ uint64_t whole_weight(double w) {   // in units of 2^-44: those are the last places of numbers from 256 to 512
    return (uint64_t)(__double_as_longlong(w + 384.0) - __double_as_longlong(384.0));
}

// the largest of a piece's values, NaN if one is
template <class E> __device__ __forceinline__ float largest(const uint4& q);
template <> __device__ __forceinline__ float largest<__half>(const uint4& q) {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
template <> __device__ __forceinline__ float largest<__nv_bfloat16>(const uint4& q) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
__device__ __forceinline__ float larger_or_nan(float p, float q) {
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(p), "f"(q));
    return v;
}
template <> __device__ __forceinline__ float largest<float>(const uint4& q) {
    return larger_or_nan(larger_or_nan(__uint_as_float(q.x), __uint_as_float(q.y)), larger_or_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
}

struct Found {
    uint32_t key;
    uint32_t equals;      // values of that key
    uint64_t before;      // sum in front of the first of them
};

// A row's filters.
struct RowFilters {
    double T, p, m, u;
    int k;
    bool by_rank, by_sum, by_size, greedy;
    __device__ __forceinline__ RowFilters(const SampleArgs& a, int64_t row) {
        T = a.T ? (double)a.T[row] : a.T_all, p = a.p ? (double)a.p[row] : a.p_all, m = a.m ? (double)a.m[row] : a.m_all, k = a.k ? a.k[row] : a.k_all;
        u = fmin(fmax((double)a.u[row], 0.0), 1.0);
        by_rank = k > 0 && k < a.V, by_sum = p < 1.0, by_size = m > 0.0, greedy = !(T > 0.0 && k != 1 && a.V > 1);
    }
    // a value below which none has a weight of m (a little too low: the weights decide)
    __device__ __forceinline__ float size_bound(float top) const {
        const float least = m >= 1.0 ? top : fminf(top, (float)fmax(-3.4e38, (double)top + T * log(m) * (1 + 1e-6)));
        return least - 1e-6f * fabsf(least);
    }
};

enum SampleState : int { SP_LOOK, SP_DONE, SP_AGAIN };   // the row has its id; it has to be done in whole numbers

// Twice what adding up a piece's weights in 32 bits may lose: eight partial sums, 35 / 8 of 2^-24 of the last one.
constexpr double ADDING = 8.75 * 0x1p-24;

// Few values of a row (key and id of each), sorted, and what they answer: by a block's first `size` threads.
struct FewShared {
    uint64_t red[32], told[2];
    uint32_t votes[2][32], n[2];
};
template <int NT>
struct Few {
    FewShared& s;
    uint64_t* lists;       // two of NT values, and two buffers
    int lane, warp, size, turn;   // (two buffers in turn for what the threads tell each other: one barrier each)
    static __device__ __forceinline__ uint64_t entry(float v, int id) { return (uint64_t)key_of(v) << 32 | (0xffffffffu - (uint32_t)id); }
    __device__ __forceinline__ bool begin(uint32_t n) {   // whether this thread takes part in work on n values
        size = n <= 32 ? 32 : 1 << (32 - __clz(n - 1)), turn = 0;
        return (int)threadIdx.x < size;
    }
    __device__ __forceinline__ void meet() {
        if (size == 32) __syncwarp();
        else asm volatile("bar.sync 1, %0;" ::"r"(size) : "memory");
    }
    __device__ __forceinline__ uint32_t vote(bool yes) {   // how many
        uint32_t n = __popc(__ballot_sync(0xffffffffu, yes));
        if (size == 32) return n;
        turn ^= 1;
        if (lane == 0) s.votes[turn][warp] = n;
        meet();
        return __reduce_add_sync(0xffffffffu, 32 * lane < size ? s.votes[turn][lane] : 0u);
    }
    __device__ __forceinline__ uint64_t tell(bool mine, uint64_t v) {   // that of the thread for which it is `mine`
        turn ^= 1;
        if (mine) s.told[turn] = v;
        meet();
        return s.told[turn];
    }
    __device__ __forceinline__ uint64_t running(uint64_t v) {   // over the threads up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        if (size == 32) return v;
        if (lane == 31) s.red[warp] = v;
        meet();
        uint64_t ahead = lane < warp ? s.red[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        return v + ahead;
    }
    // thread r's: the r-th of n <= size values, larger ones first (0 behind them)
    __device__ uint64_t sorted(const uint64_t* list, uint32_t n) {
        const uint32_t i = threadIdx.x;
        uint64_t v = i < n ? list[i] : 0;
        for (uint32_t run = 2; run <= (uint32_t)size; run *= 2)
            for (uint32_t far = run / 2; far > 0; far /= 2) {
                uint64_t other;
                if (far >= 32) {
                    turn ^= 1;
                    uint64_t* x = lists + NT * (2 + turn);
                    x[i] = v;
                    meet();
                    other = x[i ^ far];
                } else {
                    other = __shfl_xor_sync(0xffffffffu, v, far);
                }
                const bool larger = ((i & far) == 0) == ((i & run) == 0);
                v = larger == (v > other) ? v : other;
            }
        return v;
    }
    // Of the n values of a list, behind a sum `front` of all in front of them: what is kept (`ends`: with total the row's sum; under top_k
    // that of the first k is theirs), and the draw (`draws`). Sums of weights in 32 bits, as front is one and total has some, may be `off`
    // relative.
    __device__ SampleState answer(const RowFilters& f, const RowScale& r, const uint64_t* list, uint32_t n, uint64_t front, uint64_t total, double off, bool from_top, bool ends,
                                  bool draws, uint64_t& kept, int64_t* id, float* logp) {
        const uint64_t e = sorted(list, n);
        const float v = value_of((uint32_t)(e >> 32));
        const bool on = threadIdx.x < n;
        const double wd = on ? weight(r, v) : 0.0;
        const uint64_t w = whole_weight(wd), cum = front + running(w), before = cum - w;
        // Whether X = q * all is met too closely, or not at all. With front off by a and what lies between it and all by b, relative, sums
        // up to a value and X differ by (1 - q) a front - q b (all - front) more than they should; and by what the additions' own rounding
        // makes of front in one pass and in another.
        auto unsure = [&](uint64_t X, double q, uint64_t all) {
            q = fmin(fmax(q, 0.0), 1.0);
            const double slack = off * ((1.0 - q) * (double)front + q * fmax(0.0, (double)all - (double)front)) + ADDING * (double)front + 4.0;
            const bool close = on && fabs((double)cum - (double)X) <= slack, met = on && (double)cum >= (double)X + slack;
            return vote(close) != 0 || vote(met) == 0 || (!from_top && (double)front + slack >= (double)X);
        };
        if (ends) {
            uint32_t count = f.by_rank ? min((uint32_t)f.k, n) : n;
            if (f.by_rank) total = tell(threadIdx.x + 1 == count, cum);
            if (f.by_sum) {
                const uint64_t X = (uint64_t)fmax(1.0, ceil(f.p * (double)total));
                if (off > 0 && unsure(X, f.p, total)) return SP_AGAIN;
                count = min(count, vote(on && before < X));
            }
            if (f.by_size) {
                const uint32_t large = vote(on && wd >= f.m);
                if (!from_top && large < count) return SP_AGAIN;   // (the end may lie in front of these)
                count = max(1u, min(count, large));
            }
            kept = f.by_rank || f.by_sum || f.by_size ? tell(threadIdx.x + 1 == count, cum) : total;
        }
        if (draws) {
            const uint64_t X = min(kept, (uint64_t)floor(f.u * (double)kept) + 1);
            // (kept is exact where its end was found here, among values from the top; one found in another list, or the row's sum, is off,
            // and X with it)
            if (off > 0 && !(ends && from_top && (f.by_sum || f.by_size)) && unsure(X, f.u, kept)) return SP_AGAIN;
            const bool mine = on && before < X && X <= cum;
            if (mine) {
                *id = 0xffffffffu - (uint32_t)e;
                double l = -log((double)kept * (1.0 / SP_ONE));
                if (v != r.top) l += ((double)v - (double)r.top) / f.T;
                *logp = (float)l;
            }
            if (off > 0 && vote(mine) == 0) return SP_AGAIN;   // (without `off` kept is this list's: X is met)
        }
        return SP_DONE;
    }
};

template <int NT>
struct alignas(16) SampleShared {
    uint64_t cum[SP_BINS], sub[SP_SUB];
    uint32_t part[3][SP_BINS];   // sums of a weight's lowest 15 bits, the next 15, and the rest
    uint32_t list[SP_LIST], own[SP_LIST];
    double tab[16];
    uint64_t red[NT / 32], mine;
    double part_sum[2];
    uint64_t kept;
    FewShared few;
    uint32_t least, most, matches[NT / 32], matched;
    uint32_t top, tops[NT / 32];
    uint32_t digit[2], left[2], bound;    // of the search among the threads' maxima: of each pass its own
    int state;                            // what comes next: the bins of up to two brackets, or a SampleState
    int bins[4];
    Found found;
};
template <class E, int NT>
struct Sampler {
    static constexpr int PER = 16 / sizeof(E), WARPS = NT / 32;
    SampleShared<NT>& s;
    const uint4* row;      // this block's pieces, in shared memory
    int pieces, per_warp;  // of this block; of a warp: whole rounds of 32
    cg::cluster_group cluster;
    int blocks, rank;
    RowScale r;
    int lane, warp;

    __device__ __forceinline__ void join() {   // all blocks of the row
        if (blocks > 1) cluster.sync();
        else __syncthreads();
    }
    template <class T>
    __device__ __forceinline__ T* of(T* p, int other) { return blocks > 1 ? cluster.map_shared_rank(p, other) : p; }

    // f(value, piece of the warp's round) for every value of the block
    template <class F>
    __device__ __forceinline__ void each(F f) {
        const int end = min(pieces, (warp + 1) * per_warp);
        for (int c = warp * per_warp + lane; c < end; c += 32) {
            float v[PER];
            unpack<E>(row[c], v);
#pragma unroll
            for (int i = 0; i < PER; ++i) f(v[i]);
        }
    }
    template <class Op>
    __device__ __forceinline__ uint64_t reduce(uint64_t v, Op op) {   // over all threads of all blocks
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, (uint64_t)__shfl_xor_sync(0xffffffffu, v, o));
        if (lane == 0) s.red[warp] = v;
        __syncthreads();
        v = s.red[lane % WARPS];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
            if (o < WARPS) v = op(v, w);
        }
        if (blocks > 1) {
            if (threadIdx.x == 0) s.mine = v;
            cluster.sync();
            for (int b = 1; b < blocks; ++b) v = op(v, *of(&s.mine, (rank + b) % blocks));
            cluster.sync();
        } else {
            __syncthreads();
        }
        return v;
    }
    __device__ __forceinline__ void clear(int bins) {
        for (int i = threadIdx.x; i < bins; i += NT) s.part[0][i] = s.part[1][i] = s.part[2][i] = 0;
        __syncthreads();
    }
    template <bool COUNT>
    __device__ __forceinline__ void add(int bin, float v) {
        if (COUNT) {
            atomicAdd(&s.part[0][bin], 1u);
            return;
        }
        const uint64_t w = whole_weight(weight(r, v));
        if (w == 0) return;
        atomicAdd(&s.part[0][bin], (uint32_t)w & 0x7fffu);
        atomicAdd(&s.part[1][bin], (uint32_t)(w >> 15) & 0x7fffu);
        atomicAdd(&s.part[2][bin], (uint32_t)(w >> 30));
    }
    // ---- few values, in the first block
    __device__ __forceinline__ uint64_t* lists() { return reinterpret_cast<uint64_t*>(s.part[1]); }   // 4 NT of them
    __device__ __forceinline__ void keep(float v, int id, int list = 0) {
        const uint32_t at = atomicAdd(of(&s.few.n[list], 0), 1u);
        if (at < (uint32_t)NT) of(lists() + NT * list, 0)[at] = Few<NT>::entry(v, id);
    }
    // A bound that at least k of this block's threads reach with their maxima (to its upper 16 bits), or 0. Each digit by a histogram of the threads.
    // (A pass has a digit of its own: nobody waits between reading the first one's and the second pass.)
    __device__ uint32_t reached(uint32_t k, uint32_t key) {
        uint32_t bound = 0;
        if (threadIdx.x < 2) s.digit[threadIdx.x] = 256;
        for (int pass = 0; pass < 2; ++pass) {
            const int shift = 24 - 8 * pass;
            if (threadIdx.x < 256) s.part[0][threadIdx.x] = 0;
            __syncthreads();
            if (key != 0 && (shift == 24 || key >> 24 == bound >> 24)) atomicAdd(&s.part[0][key >> shift & 255], 1u);
            __syncthreads();
            if (warp == 0) {
                uint32_t n[8], sum = 0, up;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += n[i] = s.part[0][255 - 8 * lane - i];
                up = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t w = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += w;
                }
                uint32_t before = up - sum;
                if (before < k && k <= up) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (before < k && k <= before + n[i]) s.digit[pass] = 255 - 8 * lane - i, s.left[pass] = k - before;
                        before += n[i];
                    }
                }
            }
            __syncthreads();
            if (s.digit[pass] == 256) return 0;
            bound |= s.digit[pass] << shift;
            k = s.left[pass];
        }
        return bound;
    }
    // running sums of the histogram, over all blocks; every block has them. (Each adds up a share of the bins and hands it round: all of
    // them by every block took 90 us in clusters of eight.)
    template <int BINS>
    __device__ __forceinline__ void run_up(uint64_t* cum) {
        constexpr int EACH = (BINS + NT - 1) / NT;
        join();
        const int share = BINS / blocks;
        for (int bin = rank * share + threadIdx.x; bin < (rank + 1) * share; bin += NT) {
            uint64_t sum = 0;
#pragma unroll
            for (int b = 0; b < SP_MAX_BLOCKS; ++b)
                if (b < blocks) sum += (uint64_t)*of(&s.part[0][bin], b) + ((uint64_t)*of(&s.part[1][bin], b) << 15) + ((uint64_t)*of(&s.part[2][bin], b) << 30);
#pragma unroll
            for (int b = 0; b < SP_MAX_BLOCKS; ++b)
                if (b < blocks) *of(&cum[bin], b) = sum;
        }
        join();
        uint64_t v[EACH], sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int bin = threadIdx.x * EACH + i;
            if (bin < BINS) sum += cum[bin];
            v[i] = sum;
        }
        uint64_t up = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t w = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += w;
        }
        if (lane == 31) s.red[warp] = up;
        __syncthreads();
        uint64_t base = lane < warp ? s.red[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
        base += up - sum;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (threadIdx.x * EACH + i < BINS) cum[threadIdx.x * EACH + i] = base + v[i];
        __syncthreads();
    }
    template <int BINS>
    static __device__ __forceinline__ int search(const uint64_t* cum, uint64_t X) {   // the first bin that reaches X
        int lo = 0, hi = BINS - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (cum[mid] >= X) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }

    // Where the running sum over the keys above `floor_` reaches X (1 <= X <= their sum, which s.cum has): weights, or ranks (COUNT).
    template <bool COUNT>
    __device__ Found locate(uint64_t X, uint32_t floor_) {
        const int bin = search<SP_BINS>(s.cum, X);
        Found out = {0, 0, bin ? s.cum[bin - 1] : 0};
        uint32_t lo = 0, hi = 0xffffffffu;
        for (int level = 0;; ++level) {
            auto inside = [&](float v, uint32_t key) { return key > floor_ && (level ? key >= lo && key <= hi : bin_of(r, v) == bin); };
            if (threadIdx.x == 0) s.few.n[0] = 0, s.least = 0xffffffffu, s.most = 0;
            __syncthreads();
            each([&](float v) {
                const uint32_t key = key_of(v);
                if (!inside(v, key)) return;
                const uint32_t at = atomicAdd(&s.few.n[0], 1u);
                if (at < SP_LIST) s.own[at] = key;
                atomicMin(&s.least, key);
                atomicMax(&s.most, key);
            });
            join();
            uint32_t n = 0;
            lo = 0xffffffffu, hi = 0;
            for (int b = 0; b < blocks; ++b) {
                const uint32_t have = *of(&s.few.n[0], b);
                if (n + have <= SP_LIST)
                    for (uint32_t i = threadIdx.x; i < have; i += NT) s.list[n + i] = *of(&s.own[0] + i, b);
                n += have;
                lo = min(lo, *of(&s.least, b)), hi = max(hi, *of(&s.most, b));
            }
            join();
            out.key = lo, out.equals = n;
            if (lo >= hi || level > 5) return out;   // (four divisions take 32 bits apart)
            if (n <= SP_LIST) break;
            // the keys between in 1024 parts
            const int shift = max(0, 32 - __clz(hi - lo) - 10);
            clear(SP_SUB);
            each([&](float v) {
                const uint32_t key = key_of(v);
                if (key > floor_ && key >= lo && key <= hi) add<COUNT>((int)((hi - key) >> shift), v);
            });
            run_up<SP_SUB>(s.sub);
            const int part = search<SP_SUB>(s.sub, X - out.before);
            if (part) out.before += s.sub[part - 1];
            const uint32_t top = hi - ((uint32_t)part << shift);
            if (top - lo >= 1u << shift) lo = top - ((1u << shift) - 1);
            hi = top;
        }
        const uint32_t i = threadIdx.x, n = out.equals;
        if (i < n) s.sub[i] = COUNT ? 1 : whole_weight(weight(r, value_of(s.list[i])));
        __syncthreads();
        if (i < n) {
            const uint32_t key = s.list[i];
            uint64_t before = out.before;
            uint32_t equals = 0;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t other = s.list[j];
                if (other > key) before += s.sub[j];
                equals += other == key;
            }
            if (before < X && X <= before + equals * s.sub[i]) s.found = Found{key, equals, before};
        }
        __syncthreads();
        out = s.found;
        __syncthreads();
        return out;
    }
};

template <class E, int NT>
__global__ void __launch_bounds__(NT) sample_filtered_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sample_smem[];
    SampleShared<NT>& s = *reinterpret_cast<SampleShared<NT>*>(sample_smem);
    unsigned char* row_bytes = sample_smem + sizeof(SampleShared<NT>);
    constexpr int PER = 16 / sizeof(E);
    Sampler<E, NT> x = {s, reinterpret_cast<const uint4*>(row_bytes), 0, 0, cg::this_cluster()};
    x.blocks = (int)x.cluster.num_blocks(), x.rank = (int)x.cluster.block_rank();
    x.lane = threadIdx.x & 31, x.warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x / x.blocks;
    const E* logits = static_cast<const E*>(a.logits) + row * a.stride;
    const Extent all = rows_extent(a.logits, a.rows, a.stride, a.V, sizeof(E));
    // the row from its last 16-byte boundary on: the first `skip` values of the first piece are not its own
    const int skip = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(E)), all_pieces = (skip + a.V + PER - 1) / PER;
    const int first = x.rank * a.share;
    x.pieces = max(0, min(a.share, all_pieces - first));
    x.per_warp = (x.pieces + NT - 1) / NT * 32;
    if (threadIdx.x < 16) s.tab[threadIdx.x] = exp2((double)threadIdx.x / 16.0);
    if (threadIdx.x < 2) s.few.n[threadIdx.x] = 0;
    const RowFilters f = RowFilters(a, row);
    const double T = f.T, p = f.p, m = f.m, u = f.u;
    const int k = f.k;
    const bool by_rank = f.by_rank, by_sum = f.by_sum, by_size = f.by_size, greedy = f.greedy;
    const int own = x.warp * x.per_warp + x.lane, end = min(x.pieces, (x.warp + 1) * x.per_warp);   // a thread's pieces: own, own + 32 ..
    float top = -INFINITY;
    {
        uint4* to = reinterpret_cast<uint4*>(row_bytes);
        for (int c = own; c < end; c += 32) {
            const int at = (first + c) * PER - skip;   // of the row
            uint4 q;
            if (at >= 0 && at + PER <= a.V) {
                q = make_uint4(0, 0, 0, 0);
                if (all.holds(logits + at, PER)) q = __ldcs(reinterpret_cast<const uint4*>(logits + at));
            } else {
                float v[PER];
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] = at + i >= 0 && at + i < a.V && all.holds(logits + at + i) ? to_f(logits[at + i]) : -INFINITY;
                q = pack<E>(v);
            }
            to[c] = q;
            top = larger_or_nan(top, largest<E>(q));
        }
    }
    const uint32_t own_top = own < end ? (top == top ? key_of(top) : 0xffffffffu) : 0;   // 0: a thread without values; a NaN on top of all
    uint32_t key = __reduce_max_sync(0xffffffffu, own_top);
    if (x.lane == 0) s.tops[x.warp] = key;
    __syncthreads();
    key = __reduce_max_sync(0xffffffffu, s.tops[x.lane % (NT / 32)]);
    if (x.blocks > 1) {
        if (threadIdx.x == 0) s.top = key;
        x.cluster.sync();
        for (int b = 0; b < x.blocks; ++b) key = max(key, *x.of(&s.top, b));
    }
    auto larger = [](uint64_t p, uint64_t q) { return p > q ? p : q; };
    auto sum = [](uint64_t p, uint64_t q) { return p + q; };
    if (key == 0xffffffffu || key <= key_of(-INFINITY)) {   // a NaN, or nothing to draw
        if (x.rank == 0 && threadIdx.x == 0) a.ids[row] = -1, a.logp[row] = NAN;
        if (x.blocks > 1) x.cluster.sync();
        return;
    }
    top = value_of(key);
    x.r = {top, 0.f, 1.4426950408889634074 / T, s.tab};
    const int first_id = first * PER - skip;

    Few<NT> few = {s.few, x.lists(), x.lane, x.warp, 32, 0};
    uint64_t kept = 0;
    bool done = false;
    if (!greedy && ((by_rank && k <= 600 / x.blocks) || (!by_rank && !by_sum && by_size && top < INFINITY))) {
        // ---- few values
        float least;
        if (by_rank) {
            uint32_t bound = x.reached((uint32_t)k, own_top);
            if (x.blocks > 1) {   // the largest of the blocks' bounds will do
                if (threadIdx.x == 0) s.bound = bound;
                x.cluster.sync();
                for (int b = 0; b < x.blocks; ++b) bound = max(bound, *x.of(&s.bound, b));
            }
            least = bound > key_of(-INFINITY) ? value_of(bound) : -INFINITY;
        } else {
            least = f.size_bound(top);
        }
        __syncthreads();
        for (int c = own; c < end; c += 32) {
            const uint4 q = x.row[c];
            if (!(largest<E>(q) >= least)) continue;
            float v[PER];
            unpack<E>(q, v);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (v[i] >= least && v[i] > -INFINITY) x.keep(v[i], first_id + c * PER + i);
        }
        x.join();
        const uint32_t n = *x.of(&s.few.n[0], 0);
        if (n <= (uint32_t)NT) {   // (the same in all blocks)
            if (x.rank == 0 && few.begin(n)) few.answer(f, x.r, x.lists(), n, 0, 0, 0.0, true, true, true, kept, a.ids + row, a.logp + row);
            done = true;
        }
        if (x.blocks > 1) x.cluster.sync();   // (the first block's count has been read)
    } else if (!greedy && !by_rank && top < INFINITY && T > 1e-6 && T < 1e6) {
        // ---- a bracket
        constexpr double EPS = 0x1p-19;                              // of sums of weight32: 2^-22 + 2^-23 + 2^-20, and up to 2^-21 for adding up a piece's eight
        constexpr float MAGIC = 8388608.f;                           // 2^23: the last places are whole numbers
        const float c = (float)x.r.c, c_low = (float)(x.r.c - (double)c), bins = (float)(SP_BINS / (32.0 * T)), far = (SP_BINS - 1) / bins;
        for (int i = threadIdx.x; i < SP_BINS; i += NT) s.part[0][i] = 0;
        if (threadIdx.x == 0) s.state = SP_LOOK;
        __syncthreads();
        auto block_sums = [&](double v, double w, double (&out)[2]) {   // in the first block: over all blocks
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o), w += __shfl_xor_sync(0xffffffffu, w, o);
            double* r = reinterpret_cast<double*>(s.sub);
            if (x.lane == 0) r[x.warp] = v, r[32 + x.warp] = w;
            __syncthreads();
            if (x.warp < 2) {
                v = x.lane < NT / 32 ? r[32 * x.warp + x.lane] : 0.0;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (x.lane == 0) s.part_sum[x.warp] = v;
            }
            x.join();
            out[0] = out[1] = 0.0;
            if (x.rank == 0)
                for (int b = 0; b < x.blocks; ++b) out[0] += *x.of(&s.part_sum[0], b), out[1] += *x.of(&s.part_sum[1], b);
        };
        // (values beyond `far`, -inf among them, count as those there: 2^-46 each)
        double mine = 0.0, sums[2];
        for (int i = own; i < end; i += 32) {
            float v[PER], w = 0.f;
            unpack<E>(x.row[i], v);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const float d = fminf(top - v[j], far);
                atomicAdd(&s.part[0][__float_as_uint(fmaf(d, bins, MAGIC)) - __float_as_uint(MAGIC)], 1u);
                w += weight32(d, c, c_low);
            }
            mine += (double)w;
        }
        block_sums(mine, 0.0, sums);
        const double total = sums[0];
        const uint64_t whole = (uint64_t)(total * SP_ONE);
        const int share = SP_BINS / x.blocks;
        for (int bin = x.rank * share + threadIdx.x; bin < (x.rank + 1) * share; bin += NT) {   // the counts of all blocks, in the first one
            uint32_t n = 0;
#pragma unroll
            for (int o = 0; o < SP_MAX_BLOCKS; ++o)
                if (o < x.blocks) n += *x.of(&s.part[0][bin], o);
            *x.of(&s.part[1][bin], 0) = n;
        }
        x.join();
        if (x.rank == 0) {
            // Running counts, and sums of the weights as if a bin's values lay in its middle: they are off by half a bin's width each, 0.4
            // %, to either side, and so, many together, by little. That they say where to look is all that is asked of them: `answer` sees
            // whether the place was right.
            constexpr int EACH = SP_BINS / NT;
            float* run = reinterpret_cast<float*>(s.cum);
            uint32_t n[EACH], count = 0;
            float b[EACH], weights = 0.f;
            const float q = c / bins;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int bin = threadIdx.x * EACH + i;
                n[i] = s.part[1][bin];
                float w;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(-(float)bin * q));
                weights += (float)n[i] * w;
                count += n[i];
                b[i] = weights;
                n[i] = count;
            }
            float w_up = weights;
            uint32_t n_up = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float l = __shfl_up_sync(0xffffffffu, w_up, o);
                const uint32_t h = __shfl_up_sync(0xffffffffu, n_up, o);
                if (x.lane >= o) w_up += l, n_up += h;
            }
            float2* warps = reinterpret_cast<float2*>(s.red);
            if (x.lane == 31) warps[x.warp] = make_float2(w_up, __uint_as_float(n_up));
            __syncthreads();   // (and all counts have been read)
            float w_base = x.lane < x.warp ? warps[x.lane].x : 0.f;
            const uint32_t n_base = __reduce_add_sync(0xffffffffu, x.lane < x.warp ? __float_as_uint(warps[x.lane].y) : 0u) + n_up - count;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) w_base += __shfl_xor_sync(0xffffffffu, w_base, o);
            w_base += w_up - weights;
#pragma unroll
            for (int i = 0; i < EACH; ++i) run[threadIdx.x * EACH + i] = w_base + b[i], s.part[0][threadIdx.x * EACH + i] = n_base + n[i];
            __syncthreads();
            if (x.warp == 0) {   // lane 0 .. 3: the bins in which the lower and upper end of the draw's bracket lie, and of the end of what is kept
                const double X = (x.lane < 2 ? u : 1.0) * (by_sum ? p : 1.0) * total;
                const float at = (float)(x.lane & 1 ? X * 1.0015 : X * 0.9988);
                int lo = 0, hi = SP_BINS - 1;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (run[mid] >= at) hi = mid;
                    else lo = mid + 1;
                }
                int u0 = __shfl_sync(0xffffffffu, lo, 0), u1 = __shfl_sync(0xffffffffu, lo, 1), p0 = SP_BINS, p1 = SP_BINS - 1;
                if (by_sum) p0 = __shfl_sync(0xffffffffu, lo, 2), p1 = __shfl_sync(0xffffffffu, lo, 3);
                auto values = [&](int from, int to) { return s.part[0][to] - (from > 0 ? s.part[0][from - 1] : 0); };
                const int last = by_sum ? p1 : u1;
                int state = SP_LOOK;
                if (values(0, last) <= (uint32_t)NT) {           // all from the top are few enough
                    u0 = 0, u1 = last, p0 = SP_BINS;
                } else if (by_sum && values(u0, p1) <= (uint32_t)NT) {   // one bracket for both
                    u1 = p1, p0 = SP_BINS;
                } else if (values(u0, u1) > (uint32_t)NT || (by_sum && (u1 >= p0 || values(p0, p1) > (uint32_t)NT))) {
                    state = SP_AGAIN;
                }
                if (x.lane == 0) s.bins[0] = u0, s.bins[1] = u1, s.bins[2] = p0, s.bins[3] = p1, s.state = state;
            }
        }
        x.join();
        int state = *x.of(&s.state, 0);
        if (state == SP_LOOK) {
            const float u0 = MAGIC + (float)*x.of(&s.bins[0], 0), u1 = MAGIC + (float)*x.of(&s.bins[1], 0), p0 = MAGIC + (float)*x.of(&s.bins[2], 0), p1 = MAGIC + (float)*x.of(&s.bins[3], 0);
            const bool two = p0 < MAGIC + SP_BINS, from_top = u0 == MAGIC;
            double ahead = 0.0;
            mine = 0.0;
            for (int i = own; i < end; i += 32) {
                const uint4 q = x.row[i];
                if (from_top && !two && fmaf(fminf(top - largest<E>(q), far), bins, MAGIC) > u1) continue;
                float v[PER], w0 = 0.f, w1 = 0.f;
                unpack<E>(q, v);
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const float d = fminf(top - v[j], far), f = fmaf(d, bins, MAGIC);
                    if (f < u0 || (two && f < p0)) {
                        const float w = weight32(d, c, c_low);
                        w1 += w;
                        if (f < u0) w0 += w;
                    }
                    if (f >= u0 && f <= u1 && v[j] > -INFINITY) x.keep(v[j], first_id + i * PER + j);
                    else if (two && f >= p0 && f <= p1 && v[j] > -INFINITY) x.keep(v[j], first_id + i * PER + j, 1);
                }
                mine += (double)w0, ahead += (double)w1;
            }
            block_sums(mine, ahead, sums);
            if (x.rank == 0) {
                const uint32_t n0 = s.few.n[0], n1 = s.few.n[1];
                const uint64_t front = from_top ? 0 : (uint64_t)(sums[0] * SP_ONE);
                state = n0 <= (uint32_t)NT && n1 <= (uint32_t)NT ? SP_DONE : SP_AGAIN;
                if (two && state == SP_DONE) {
                    if (few.begin(n1)) state = few.answer(f, x.r, x.lists() + NT, n1, (uint64_t)(sums[1] * SP_ONE), whole, EPS, false, true, false, kept, nullptr, nullptr);
                    if (threadIdx.x == 0) s.state = state, s.kept = kept;
                    __syncthreads();
                    state = s.state, kept = s.kept;
                    __syncthreads();
                }
                if (state == SP_DONE && few.begin(n0))
                    state = few.answer(f, x.r, x.lists(), n0, front, whole, EPS, from_top, !two, true, kept, a.ids + row, a.logp + row);
                if (threadIdx.x == 0) s.state = state;
            }
            x.join();
            state = *x.of(&s.state, 0);
        }
        done = state == SP_DONE;
        x.join();   // (the first block's word has been read)
    }
    if (done) return;

    // ---- whole numbers
    uint64_t ordinal = 0;
    double logp = 0.0;
    if (!greedy) {
        float low = INFINITY;
        x.each([&](float v) {
            if (v > -INFINITY) low = fminf(low, v);
        });
        low = value_of(~(uint32_t)x.reduce((uint64_t)~key_of(low), larger));
        const float range = (float)fmin(32.0 * T, (double)top - (double)low);
        x.r.bins = range > 0.f ? SP_BINS / range : 0.f;
        uint32_t floor_ = 0;       // keys above this one count (0 is no value's)
        uint64_t ties = 0, tied = 0;
        if (by_rank) {
            x.clear(SP_BINS);
            x.each([&](float v) { x.template add<true>(bin_of(x.r, v), v); });
            x.template run_up<SP_BINS>(s.cum);
            const Found f = x.template locate<true>((uint64_t)k, 0);
            floor_ = f.key;
            ties = (uint64_t)k - f.before;
            tied = whole_weight(weight(x.r, value_of(floor_)));
        }
        x.clear(SP_BINS);
        x.each([&](float v) {
            if (key_of(v) > floor_) x.template add<false>(bin_of(x.r, v), v);
        });
        x.template run_up<SP_BINS>(s.cum);
        const uint64_t above = s.cum[SP_BINS - 1];
        kept = above + ties * tied;
        uint32_t last = floor_;    // key of the last value that is kept, where a filter has set one
        // the front part that reaches X ends at ...
        auto reach = [&](uint64_t X, uint64_t& before, uint64_t& w) {
            if (X > above) {
                before = above, w = tied;
                return floor_;
            }
            const Found f = x.template locate<false>(X, floor_);
            before = f.before, w = whole_weight(weight(x.r, value_of(f.key)));
            return f.key;
        };
        if (by_sum) {
            const uint64_t X = min(kept, (uint64_t)fmax(1.0, ceil(p * (double)kept)));
            uint64_t before, w;
            last = reach(X, before, w);
            kept = before + (X - before + w - 1) / w * w;
        }
        if (by_size && !(last != 0 && weight(x.r, value_of(last)) >= m)) {
            const double far = 1e-6 - log2(m);   // (a little too far)
            uint64_t mine = 0;
            x.each([&](float v) {
                if (key_of(v) <= floor_ || !(v == top || ((double)top - (double)v) * x.r.c <= far)) return;
                const double w = weight(x.r, v);
                if (w >= m) mine += whole_weight(w);
            });
            kept = max(SP_ONE, min(kept, x.reduce(mine, sum)));
        }
        const uint64_t X = min(kept, (uint64_t)floor(u * (double)kept) + 1);
        uint64_t before, w;
        key = reach(X, before, w);
        ordinal = (X - before + w - 1) / w - 1;
        logp = -log((double)kept * (1.0 / SP_ONE));
        if (value_of(key) != top) logp += ((double)value_of(key) - (double)top) / T;
    }
    // the value of that key with `ordinal` of them in front of it
    uint32_t matches = 0;
    x.each([&](float v) { matches += key_of(v) == key; });
    matches = __reduce_add_sync(0xffffffffu, matches);
    if (x.lane == 0) s.matches[x.warp] = matches;
    __syncthreads();
    uint32_t before = 0, in_block = 0;
    for (int i = 0; i < NT / 32; ++i) {
        if (i < x.warp) before += s.matches[i];
        in_block += s.matches[i];
    }
    if (x.blocks > 1) {
        if (threadIdx.x == 0) s.matched = in_block;
        x.cluster.sync();
        for (int b = 0; b < x.rank; ++b) before += *x.of(&s.matched, b);
        x.cluster.sync();
    }
    if (ordinal < before || ordinal >= (uint64_t)before + matches) return;
    for (int c0 = x.warp * x.per_warp; c0 < end; c0 += 32) {
        const int c = c0 + x.lane;
        uint32_t mask = 0;
        if (c < end) {
            float v[PER];
            unpack<E>(x.row[c], v);
#pragma unroll
            for (int i = 0; i < PER; ++i) mask |= (uint32_t)(key_of(v[i]) == key) << i;
        }
        const uint32_t n = __popc(mask);
        uint32_t up = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t w = __shfl_up_sync(0xffffffffu, up, o);
            if (x.lane >= o) up += w;
        }
        const uint32_t from = before + up - n;
        if (ordinal >= from && ordinal < from + n) {
            for (uint32_t i = from; i < ordinal; ++i) mask &= mask - 1;
            a.ids[row] = (int64_t)(first + c) * PER - skip + __ffs(mask) - 1;
            a.logp[row] = (float)logp;
        }
        before += __shfl_sync(0xffffffffu, up, 31);
    }
}

// ---- 16-bit logits: one counter for each of their 65536 values --------------------------------------------------------------------------
// A row's histogram over the values themselves, in shared memory, says everything but which id has a value: what is kept and drawn is found
// among the counters, whose running sums are exact, and the row is read once more (from L2) for the id. No value of the row needs an
// exponential: the counters do, and eight of them that follow one another, a unit, whose values are equally far apart, need one of them and
// its products with exp(-distance / T). Where the filters leave few values (a small top-k; min-p by itself), only those are gathered that
// reach a bound: some k of the threads' own maxima do, and so do k values. What bounds it: for rows that wait for an SM the atomics (3.3
// cycles for a warp's: two of its values meet a bank), the units' weights, and the row read twice; for the only row of an SM the steps
// behind one another, each by code that has to be fetched. fp16, 65536 values, on several boxes: one row 21 to 23 us under top-p 0.7 (8 to
// 17 under min-p 0.05), 320 rows with filters of their own 43 to 57, in three turns of 148; 37 x 50277 bf16 16 to 18.5. In clusters that
// take exponentials and search (as fp32 rows do, above) the 320 rows took 109.
//
// Counters lie in the order of the values, larger ones first, eight in 16 bytes. Eight units are a group, whose sums are run up over the
// block; a question is answered by a search among them and by the 64 counters of one group, by the first warp.
//
// A counter holds up to 65535: the row's last value is added when the others are counted, so that only a row of 65536 equal ones exceeds it
// (`extra`).
constexpr int SK_NT = 1024, SK_BINS = 65536, SK_GROUPS = SK_BINS / 64;
// Few values' sorting costs what k does, counting the same for all. Top-k 320 and 400 sorted, and counted: 1 x 65536 17.0, 21.1 and 19.8
// us; 1 x 32003 14.7, 18.8 and 15.0; 1 x 5003 14.7, 14.7 and 12.7 (256: 12.7); 512 x 65536 64.6, 81.3 and 72.3; 512 x 32003 51.8, 68.2 and
// 58.0; 512 x 5003 43.4, 53.6 and 45.4.
constexpr int SK_MOST_K = 320;
static_assert(SK_GROUPS == SK_NT, "a thread per group");

template <class E> struct KeyType;   // how a type's 16 bits are ordered
template <> struct KeyType<__half> {
    static constexpr int NEG_INF = 0xfc00, MANTISSA = 10, EXPONENTS = 32, LEAST = -24;   // bin of -inf (NaNs lie behind it, and in front of the other infinity); 2^LEAST is the smallest value
    static __device__ __forceinline__ uint32_t same(uint32_t two, uint32_t as) {   // 16 bits of ones where equal (0 and -0 are)
        return __heq2_mask(*reinterpret_cast<const __half2*>(&two), *reinterpret_cast<const __half2*>(&as));
    }
};
template <> struct KeyType<__nv_bfloat16> {
    static constexpr int NEG_INF = 0xff80, MANTISSA = 7, EXPONENTS = 256, LEAST = -133;
    static __device__ __forceinline__ uint32_t same(uint32_t two, uint32_t as) {
        return __heq2_mask(*reinterpret_cast<const __nv_bfloat162*>(&two), *reinterpret_cast<const __nv_bfloat162*>(&as));
    }
};
__device__ __forceinline__ uint32_t bits_of_bin(uint32_t bin) { return bin < 0x8000u ? 0x7fffu - bin : bin; }
__device__ __forceinline__ uint32_t bin_of_bits(uint32_t bits) { return bits == 0x8000u ? 0x7fffu : bits < 0x8000u ? 0x7fffu - bits : bits; }

struct alignas(16) KeyShared {
    uint4 counts[SK_BINS / 8];   // (or the lists of few values)
    uint64_t sums[SK_GROUPS];
    double step[256][9];         // exp(-j * (distance of two neighbours) / T), by their exponent (nine: lanes of other exponents meet other banks)
    unsigned short units[SK_BINS / 8];   // those with a counter in use
    uint64_t red[32];
    double tab[16], log_kept;
    FewShared few;
    uint32_t tops[32], matches[32];
    uint32_t extra, bin, n_units;
    uint64_t ties, tied, ordinal, kept;
};

template <class E>
__global__ void __launch_bounds__(SK_NT, 1) sample_keys_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char key_smem[];
    KeyShared& s = *reinterpret_cast<KeyShared*>(key_smem);
    using K = KeyType<E>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const E* logits = static_cast<const E*>(a.logits) + row * a.stride;
    const Extent all = rows_extent(a.logits, a.rows, a.stride, a.V, 2);
    // the row from its last 16-byte boundary on, as pieces of eight values; a warp's pieces follow one another
    const int skip = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / 2), pieces = (skip + a.V + 7) / 8;
    const int per_warp = (pieces + SK_NT - 1) / SK_NT * 32, own = warp * per_warp + lane, end = min(pieces, (warp + 1) * per_warp);
    auto piece = [&](int c) {   // (values outside of the row: -inf)
        const int at = c * 8 - skip;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (at >= 0 && at + 8 <= a.V) {
            if (all.holds(logits + at, 8)) q = __ldg(reinterpret_cast<const uint4*>(logits + at));
        } else {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = at + i >= 0 && at + i < a.V && all.holds(logits + at + i) ? to_f(logits[at + i]) : -INFINITY;
            q = pack<E>(v);
        }
        return q;
    };
    // Three pieces of a thread under way. (All eight at once make eight times the code of what is done with one, and the fetching of
    // instructions, which run once a row here, was what the kernel waited for most: 1 x 65536 23.7 us against 21.0, 320 x 65536 48.4
    // against 42.7.)
    uint4 q[3];
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (own + 32 * j < end) q[j] = piece(own + 32 * j);
    const RowFilters f = RowFilters(a, row);
    if (row + a.ahead < a.rows) {   // a row that a block will take when this one is done
        const char* next = reinterpret_cast<const char*>(static_cast<const E*>(a.logits) + (row + a.ahead) * a.stride) + (size_t)threadIdx.x * 128;
        if ((int64_t)threadIdx.x * 64 < a.V) asm volatile("prefetch.global.L2 [%0];" ::"l"(next));
    }
    const bool bounded = f.by_rank ? f.k <= SK_MOST_K : !f.by_sum && f.by_size, counting = !f.greedy && !bounded;
    uint32_t* words = reinterpret_cast<uint32_t*>(s.counts);
    auto count = [&](uint32_t bin) { atomicAdd(words + (bin >> 1), bin & 1 ? 0x10000u : 1u); };
    auto clear = [&]() {
        for (int i = threadIdx.x; i < SK_BINS / 8; i += SK_NT) s.counts[i] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x == 0) s.extra = 0;
        if (threadIdx.x < K::EXPONENTS) {
            const double one = exp(-scalbn(1.0, max((int)threadIdx.x, 1) - 1 + K::LEAST) / f.T);
            double w = 1.0;
#pragma unroll
            for (int j = 0; j < 8; ++j, w *= one) s.step[threadIdx.x][j] = w;
        }
    };
    auto count_piece = [&](const uint4& q, int c) {
        const int at = c * 8 - skip;
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        if (at >= 0 && at + 8 < a.V) {   // (the row's last value is added below)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t sign = (w[i] >> 15) & 0x00010001u, bins = w[i] ^ (0x7fff7fffu - sign * 0x7fffu);
                count(bins & 0xffffu);
                count(bins >> 16);
            }
        } else {
#pragma unroll 1
            for (int i = max(0, -at); i < 8 && at + i < a.V - 1; ++i) {
                const uint32_t two = i < 2 ? w[0] : i < 4 ? w[1] : i < 6 ? w[2] : w[3], bits = two >> (16 * (i & 1)) & 0xffffu;
                count(bits < 0x8000u ? 0x7fffu - bits : bits);
            }
        }
    };
    if (threadIdx.x < 16) s.tab[threadIdx.x] = exp2((double)threadIdx.x / 16.0);
    if (threadIdx.x < 2) s.few.n[threadIdx.x] = 0;
    if (counting) {
        clear();
        __syncthreads();
    }
    float top = -INFINITY;
#pragma unroll 1
    for (int c = own; c < end; c += 32) {
        const uint4 v = q[0];
        q[0] = q[1], q[1] = q[2];
        if (c + 96 < end) q[2] = piece(c + 96);
        top = larger_or_nan(top, largest<E>(v));
        if (counting) count_piece(v, c);
    }
    constexpr int AHEAD = 8;   // of the passes behind this one
    const uint32_t own_top = own < end ? (top == top ? key_of(top) : 0xffffffffu) : 0;   // a NaN on top of all
    uint32_t top_key = __reduce_max_sync(0xffffffffu, own_top);
    if (lane == 0) s.tops[warp] = top_key;
    __syncthreads();
    top_key = __reduce_max_sync(0xffffffffu, s.tops[lane]);
    if (top_key == 0xffffffffu || top_key <= key_of(-INFINITY)) {   // a NaN, or nothing to draw
        if (threadIdx.x == 0) a.ids[row] = -1, a.logp[row] = NAN;
        return;
    }
    auto bin_at = [&](float v) {
        const E t = from_f<E>(v);
        return bin_of_bits(*reinterpret_cast<const unsigned short*>(&t));
    };
    auto value_at = [&](uint32_t bin) { return to_f(from_bits<E>((unsigned short)bits_of_bin(bin))); };
    const float own_largest = top;
    top = value_of(top_key);
    const RowScale r = {top, 0.f, 1.4426950408889634074 / f.T, s.tab};
    if (bounded && !f.greedy) {
        // ---- few values
        float least = -INFINITY;
        if (f.by_rank) {   // The largest of 16 bits that k threads' maxima reach, digit by digit; a little more than k will do.
            const uint32_t mine = own < end ? 0xffffu - bin_at(own_largest) : 0;
            uint32_t bound = 0;
            for (int bit = 15; bit >= 0; --bit) {
                const uint32_t t = bound | 1u << bit;
                const int n = __syncthreads_count(mine >= t);
                if (n < f.k) continue;
                bound = t;
                if (n <= f.k + f.k / 8 + 16) break;
            }
            if (bound > 0xffffu - K::NEG_INF) least = value_at(0xffffu - bound);
        } else if (top < INFINITY) {
            least = f.size_bound(top);
        }
        Few<SK_NT> few = {s.few, reinterpret_cast<uint64_t*>(s.counts), lane, warp, 32, 0};
        for (int c0 = own; c0 < end && own_largest >= least; c0 += 32 * AHEAD) {   // (from L2, by the few threads that have some)
            uint4 q[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (c0 + 32 * j < end) q[j] = piece(c0 + 32 * j);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int c = c0 + 32 * j;
                if (c >= end || !(largest<E>(q[j]) >= least)) continue;
                float v[8];
                unpack<E>(q[j], v);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (v[i] >= least && v[i] > -INFINITY) {
                        const uint32_t at = atomicAdd(&s.few.n[0], 1u);
                        if (at < (uint32_t)SK_NT) few.lists[at] = few.entry(v[i], c * 8 - skip + i);
                    }
            }
        }
        __syncthreads();
        const uint32_t n = s.few.n[0];
        uint64_t kept = 0;
        if (n <= (uint32_t)SK_NT) {
            if (few.begin(n)) few.answer(f, r, few.lists, n, 0, 0, 0.0, true, true, true, kept, a.ids + row, a.logp + row);
            return;
        }
        __syncthreads();
        clear();   // (many equals, or a small min_p)
        __syncthreads();
#pragma unroll 1
        for (int c = own; c < end; c += 32) count_piece(piece(c), c);
        __syncthreads();
    }
    const uint32_t top_bin = bin_at(top);
    uint32_t bin = top_bin;
    uint64_t ordinal = 0;
    if (!f.greedy) {
        if (threadIdx.x == 0) {   // -0 is 0, and the last value
            const uint32_t minus = words[0x4000] & 0xffffu;
            words[0x4000] -= minus;
            words[0x3fff] += minus << 16;
            const uint32_t last = bin_of_bits(*reinterpret_cast<const unsigned short*>(logits + a.V - 1)), shift = 16 * (last & 1);
            if ((words[last >> 1] >> shift & 0xffffu) == 0xffffu) s.extra = 1;
            else words[last >> 1] += 1u << shift;
        }
        __syncthreads();
        const uint32_t extra = s.extra;
        auto counted = [&](uint32_t word, int half) {
            const uint32_t n = half ? word >> 16 : word & 0xffffu;
            return n == 0xffffu ? n + extra : n;
        };
        // The weight of a bin's value, from that of its unit's first (of the largest value in its unit). One way for all who ask: sums are
        // to agree to the last unit.
        auto base_of = [&](uint32_t bin) { return max(bin & ~7u, top_bin); };
        auto steps = [&](uint32_t bin) { return s.step[bits_of_bin(bin) >> K::MANTISSA & (K::EXPONENTS - 1)]; };
        auto weight_at = [&](uint32_t bin) {
            const uint32_t base = base_of(bin);
            return weight(r, value_at(base)) * steps(bin)[bin - base & 7u];   // (1 times 1 for the largest value)
        };
        // s.sums: of the groups from that of the largest value on (group g: units 8 g .. 8 g + 7), filled by run_counts or run_weights,
        // then run up over all of them.
        const int first = (int)(top_bin >> 6);
        auto run_up = [&]() {
            uint64_t v = s.sums[threadIdx.x];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t w = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += w;
            }
            if (lane == 31) s.red[warp] = v;
            __syncthreads();
            uint64_t before = lane < warp ? s.red[lane] : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
            s.sums[threadIdx.x] = v + before;
            __syncthreads();
        };
        // Where the running sum reaches X (by one warp). `one`: of two neighbouring counters and the first one's bin. Bins from `floor_` on
        // do not count.
        struct At {
            uint32_t bin;
            uint64_t before, one;   // one: what a value of the bin adds
        };
        struct Two {
            uint64_t a, b;
        };
        auto reach = [&](uint64_t X, uint32_t floor_, auto one) {
            // the group: 32 of the sums at a time
            int lo = min(__popc(__ballot_sync(0xffffffffu, s.sums[lane * 32 + 31] < X)), 31) * 32;
            lo = min(lo + __popc(__ballot_sync(0xffffffffu, s.sums[lo + lane] < X)), SK_GROUPS - 1 - first);
            const uint32_t word = words[(first + lo) * 32 + lane], b = (first + lo) * 64 + 2 * lane;   // this lane's two counters
            const uint32_t n0 = b < floor_ ? counted(word, 0) : 0, n1 = b + 1 < floor_ ? counted(word, 1) : 0;
            const Two w = one(b);
            const uint64_t v0 = n0 * w.a, v1 = n1 * w.b;
            uint64_t up = v0 + v1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t w = __shfl_up_sync(0xffffffffu, up, o);
                if (lane >= o) up += w;
            }
            up += lo ? s.sums[lo - 1] : 0;
            const int at = __ffs(__ballot_sync(0xffffffffu, up >= X)) - 1;
            const bool second = up - v1 < X;
            At out;
            out.bin = __shfl_sync(0xffffffffu, b + second, at & 31);
            out.before = __shfl_sync(0xffffffffu, second ? up - v1 : up - v1 - v0, at & 31);
            out.one = __shfl_sync(0xffffffffu, second ? w.b : w.a, at & 31);
            return out;
        };
        // how many values of w make d, at least one: by a quotient that is off by one at most
        auto how_many = [](uint64_t d, uint64_t w) {
            uint64_t n = (uint64_t)__fdividef((float)d, (float)w);
            while (n * w < d) ++n;
            while (n > 1 && (n - 1) * w >= d) --n;
            return n < 1 ? 1 : n;
        };
        uint32_t floor_ = K::NEG_INF;     // bins from here on are not kept, or have no weight
        uint64_t ties = 0, tied = 0;
        if (f.by_rank) {
            const int group = threadIdx.x;   // (one of a thread's own)
            uint32_t n = 0;
            if (first + group < SK_GROUPS)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint4 q = s.counts[(first + group) * 8 + (j + lane & 7)];   // (lanes of a warp begin at different banks)
                    n = __dp2a_lo(q.x, 0x0101u, n), n = __dp2a_lo(q.y, 0x0101u, n), n = __dp2a_lo(q.z, 0x0101u, n), n = __dp2a_lo(q.w, 0x0101u, n);
                }
            s.sums[group] = extra && n ? (uint32_t)a.V : n;
            run_up();
            if (warp == 0) {
                const At at = reach((uint64_t)f.k, SK_BINS, [](uint32_t) { return Two{1, 1}; });
                const bool weighs = at.bin < (uint32_t)K::NEG_INF;
                const uint64_t w = weighs ? whole_weight(weight_at(at.bin)) : 0;
                if (lane == 0) s.bin = weighs ? at.bin : K::NEG_INF, s.ties = weighs ? (uint64_t)f.k - at.before : 0, s.tied = w;
            }
            __syncthreads();
            floor_ = s.bin, ties = s.ties, tied = s.tied;
        }
        auto weights = [&](uint32_t b) {   // (two neighbours are of one unit)
            const uint32_t base = base_of(b);
            const double w = weight(r, value_at(base));
            const double* step = steps(b);
            return Two{whole_weight(w * step[b - base & 7u]), whole_weight(w * step[b + 1 - base & 7u])};   // (in front of the largest value: of no counter)
        };
        // The units in use, one behind the other (of 8192, some 2500 for fp16 and a few hundred for bf16), then their weights.
        __syncthreads();   // (s.sums)
        s.sums[threadIdx.x] = 0;
        if (threadIdx.x == 0) s.n_units = 0;
        __syncthreads();
        const int to_unit = ((int)floor_ + 7) / 8;
        for (int u0 = (int)(top_bin >> 3) & ~(SK_NT - 1); u0 < to_unit; u0 += SK_NT) {
            const int unit = u0 + (int)threadIdx.x;
            const uint4 q = s.counts[unit];
            const bool used = unit < to_unit && (q.x | q.y | q.z | q.w) != 0;
            const uint32_t mask = __ballot_sync(0xffffffffu, used);
            uint32_t at = 0;
            if (lane == 0 && mask) at = atomicAdd(&s.n_units, __popc(mask));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(mask & ((1u << lane) - 1));
            if (used) s.units[at] = (unsigned short)unit;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < s.n_units; i += SK_NT) {
            const uint32_t unit = s.units[i], b = unit * 8, base = base_of(b), off = base - b;
            const uint4 q = s.counts[unit];
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
            const double first_ = weight(r, value_at(base));
            const double* step = steps(b);
            uint64_t v = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t n = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
                if (b + j < floor_) v += n * whole_weight(first_ * step[j - off & 7u]);
            }
            if (extra && top_bin < floor_) v += SP_ONE;   // (the only bin in use is the largest value's)
            if (v) atomicAdd(reinterpret_cast<unsigned long long*>(&s.sums[(b >> 6) - first]), (unsigned long long)v);
        }
        __syncthreads();
        run_up();
        // The ends of what is kept, and the draw: by the first warp. The second one takes the logarithm meanwhile.
        auto hand_over = [] { asm volatile("bar.sync 2, 64;" ::: "memory"); };
        if (warp == 1) {
            hand_over();
            const double l = log((double)s.kept * (1.0 / SP_ONE));
            if (lane == 0) s.log_kept = l;
        }
        if (warp == 0) {
            const uint64_t above = s.sums[SK_GROUPS - 1];
            uint64_t kept = above + ties * tied, before, w;
            uint32_t last = ties ? floor_ : SK_BINS;   // bin of the last value that is kept, where a filter has set one
            auto ends = [&](uint64_t X) {              // the bin in which the front part that reaches X ends; what lies in front of it; its weight
                uint32_t b = floor_;
                before = above, w = tied;
                if (X <= above) {
                    const At at = reach(X, floor_, weights);
                    b = at.bin, before = at.before, w = at.one;
                }
                return b;
            };
#pragma unroll 1
            for (int step = f.by_sum ? 0 : 1; step < 2; ++step) {   // where top-p ends; then the draw (one code for both)
                if (step == 1) {
                    if (f.by_size && !(last < SK_BINS && weight_at(last) >= f.m)) {
                        // the last bin whose weight is m or more lies near this one; weights fall from bin to bin
                        const int near = (int)bin_at(top < INFINITY ? fminf(top, (float)fmax(-3.4e38, (double)top + f.T * log(f.m))) : top), b = near - 15 + lane;
                        const bool large = b < (int)top_bin || (b < K::NEG_INF && weight_at((uint32_t)b) >= f.m);
                        const int to = near - 16 + __popc(__ballot_sync(0xffffffffu, large));
                        uint64_t sum = 0;   // up to that bin
                        if (to >= (int)top_bin) {
                            const int g = to >> 6;
                            const uint32_t word = words[g * 32 + lane], c = g * 64 + 2 * lane;
                            const Two v = weights(c);
                            if (c < floor_ && (int)c <= to) sum += counted(word, 0) * v.a;
                            if (c + 1 < floor_ && (int)c + 1 <= to) sum += counted(word, 1) * v.b;
#pragma unroll
                            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                            sum += g > first ? s.sums[g - first - 1] : 0;
                        }
                        kept = max(SP_ONE, min(kept, sum));
                    }
                    if (lane == 0) s.kept = kept;
                    hand_over();
                }
                const uint64_t X = min(kept, step ? (uint64_t)floor(f.u * (double)kept) + 1 : (uint64_t)fmax(1.0, ceil(f.p * (double)kept)));
                const uint32_t b = ends(X);
                const uint64_t n = how_many(X - before, w);
                if (step == 0) last = b, kept = before + n * w;
                else if (lane == 0) s.bin = b, s.ordinal = n - 1;
            }
        }
        __syncthreads();
        bin = s.bin, ordinal = s.ordinal;
    }
    // the value of that bin with `ordinal` of them in front of it
    const uint32_t as = bits_of_bin(bin) * 0x00010001u;
    uint32_t n = 0, masks[3] = {0, 0, 0};   // a bit for each of a piece's values, eight pieces and one
    for (int i = 0, c0 = own; i == 0 || c0 < end; c0 += 32 * AHEAD, ++i) {
        uint4 q[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (c0 + 32 * j < end) q[j] = piece(c0 + 32 * j);
        if (i == 0 && threadIdx.x == 0)
            a.logp[row] = f.greedy ? 0.f : (float)((bin != top_bin ? ((double)value_at(bin) - (double)top) * (r.c * 0.693147180559945309417) : 0.0) - s.log_kept);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (c0 + 32 * j < end) {
                const uint32_t w[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
                uint32_t mask = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) mask |= (K::same(w[e], as) & 0x00020001u) << (2 * e);   // (bits 0 and 17)
                mask = (mask | mask >> 16) & 0xffu;
                n += __popc(mask);
                if (i == 0) masks[j / 4] |= mask << (8 * (j & 3));
                else masks[2] = mask;   // (j is 0)
            }
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s.matches[warp] = n;
    __syncthreads();
    uint32_t ahead = __reduce_add_sync(0xffffffffu, lane < warp ? s.matches[lane] : 0u);
    if (ordinal < ahead || ordinal >= (uint64_t)ahead + n) return;
    for (int i = 0; 32 * i < per_warp; ++i) {
        uint32_t mask = (i < 4 ? masks[0] : i < 8 ? masks[1] : masks[2]) >> (8 * (i & 3)) & 0xffu, up = __popc(mask);
        const uint32_t mine = up;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += v;
        }
        const uint32_t from = ahead + up - mine;
        if (ordinal >= from && ordinal < from + mine) {
            for (uint32_t e = from; e < ordinal; ++e) mask &= mask - 1;
            a.ids[row] = (int64_t)(own + 32 * i) * 8 - skip + __ffs(mask) - 1;
        }
        ahead += __shfl_sync(0xffffffffu, up, 31);
    }
}
// ---- top-k of the same small k for every row --------------------------------------------------------------------------------------------
// Rows are streamed, two blocks of 512 threads to an SM (k up to 256; one of 1024 up to 600), so that one reads while the other sorts: a
// row's largest values per thread, a bound that k threads reach, then only the values of a thread that reach it once more (from L2), and
// what the few values answer. Where more values than threads reach the bound (equals, mostly), the k-th largest key is searched by
// counting, and of its equals the first ids are taken. What bounds it: latency. A block loads nothing while it searches its bound (up to 16
// barriers) and sorts, and two of them to an SM read at 37 % of the memory's rate. 512 x 65536 fp32, top-k 50: 41 to 45 us on several boxes
// (3 TB/s); in clusters that keep rows in shared memory 109. For one fp32 row it takes 15 us where those take 15.5 (k 50), and 23 where
// they take 49 (k 400), of 32003 values 12.6 and 14.7, 18.8 and 44.9, of 5003 8.6 and 10.9, 16.7 and 33.6: one kernel for every number of
// rows. (Those are ahead at k 600 from some 150 rows of 32003 on: 33 us against 25.)
constexpr int ST_BATCH = 8, ST_MOST_K = 600;

template <int ST_NT>
struct alignas(16) TopShared {
    uint64_t lists[4 * ST_NT];
    FewShared few;
    double tab[16];
    uint32_t tops[32], counts[2][32];
};
template <class E, int ST_NT>
__global__ void __launch_bounds__(ST_NT, 1024 / ST_NT) sample_top_kernel(const SampleArgs a) {
    __shared__ TopShared<ST_NT> s;
    constexpr int PER = 16 / sizeof(E);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const E* logits = static_cast<const E*>(a.logits) + row * a.stride;
    const Extent all = rows_extent(a.logits, a.rows, a.stride, a.V, sizeof(E));
    const int skip = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(E)), pieces = (skip + a.V + PER - 1) / PER;
    auto piece = [&](int c) {   // (values outside of the row: -inf)
        const int at = c * PER - skip;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (at >= 0 && at + PER <= a.V) {
            if (all.holds(logits + at, PER)) q = __ldg(reinterpret_cast<const uint4*>(logits + at));
        } else {
            float v[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = at + i >= 0 && at + i < a.V && all.holds(logits + at + i) ? to_f(logits[at + i]) : -INFINITY;
            q = pack<E>(v);
        }
        return q;
    };
    RowFilters f = RowFilters(a, row);
    if (f.greedy) f.T = 1.0, f.k = 1, f.by_rank = true;   // (the first of the largest)
    if (threadIdx.x < 16) s.tab[threadIdx.x] = exp2((double)threadIdx.x / 16.0);
    if (threadIdx.x == 0) s.few.n[0] = 0;
    float largest_of[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // of this thread's batches (the last one's and all behind it)
    for (int b = 0, c0 = threadIdx.x; c0 < pieces; ++b, c0 += ST_NT * ST_BATCH) {
        uint4 q[ST_BATCH];
#pragma unroll
        for (int j = 0; j < ST_BATCH; ++j)
            if (c0 + j * ST_NT < pieces) q[j] = piece(c0 + j * ST_NT);
        float t = -INFINITY;
#pragma unroll
        for (int j = 0; j < ST_BATCH; ++j)
            if (c0 + j * ST_NT < pieces) t = larger_or_nan(t, largest<E>(q[j]));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j == min(b, 3)) largest_of[j] = larger_or_nan(largest_of[j], t);
    }
    float top = larger_or_nan(larger_or_nan(largest_of[0], largest_of[1]), larger_or_nan(largest_of[2], largest_of[3]));
    const uint32_t own_top = (int)threadIdx.x < pieces ? (top == top ? key_of(top) : 0xffffffffu) : 0;   // a NaN on top of all
    uint32_t top_key = __reduce_max_sync(0xffffffffu, own_top);
    if (lane == 0) s.tops[warp] = top_key;
    __syncthreads();
    top_key = __reduce_max_sync(0xffffffffu, s.tops[lane % (ST_NT / 32)]);
    if (top_key == 0xffffffffu || top_key <= key_of(-INFINITY)) {   // a NaN, or nothing to draw
        if (threadIdx.x == 0) a.ids[row] = -1, a.logp[row] = NAN;
        return;
    }
    top = value_of(top_key);
    const RowScale r = {top, 0.f, 1.4426950408889634074 / f.T, s.tab};
    const uint32_t none = key_of(-INFINITY) + 1;   // the least key that counts
    uint32_t bound = 0;
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | 1u << bit;
        const int n = __syncthreads_count(own_top >= t);
        if (n < f.k) continue;
        bound = t;
        if (n <= f.k + f.k / 8 + 16) break;
    }
    bound = max(bound, none);
    auto gather = [&](uint32_t bound) {   // all of its key and more
        const float least = value_of(bound);
        for (int b = 0, c0 = threadIdx.x; c0 < pieces; ++b, c0 += ST_NT * ST_BATCH) {
            const float t = b == 0 ? largest_of[0] : b == 1 ? largest_of[1] : b == 2 ? largest_of[2] : largest_of[3];
            if (!(t >= least)) continue;
            uint4 q[ST_BATCH];
#pragma unroll
            for (int j = 0; j < ST_BATCH; ++j)
                if (c0 + j * ST_NT < pieces) q[j] = piece(c0 + j * ST_NT);
#pragma unroll
            for (int j = 0; j < ST_BATCH; ++j) {
                const int c = c0 + j * ST_NT;
                if (c >= pieces || !(largest<E>(q[j]) >= least)) continue;
                float v[PER];
                unpack<E>(q[j], v);
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (v[i] >= least) {
                        const uint32_t at = atomicAdd(&s.few.n[0], 1u);
                        if (at < (uint32_t)ST_NT) s.lists[at] = Few<ST_NT>::entry(v[i], c * PER - skip + i);
                    }
            }
        }
        __syncthreads();
        return s.few.n[0];
    };
    uint32_t n = gather(bound);
    if (n > (uint32_t)ST_NT) {
        __syncthreads();   // (the count has been read)
        int turn = 0;
        auto sum = [&](uint32_t v) {   // over the block
            turn ^= 1;
            v = __reduce_add_sync(0xffffffffu, v);
            if (lane == 0) s.counts[turn][warp] = v;
            __syncthreads();
            return __reduce_add_sync(0xffffffffu, lane < ST_NT / 32 ? s.counts[turn][lane] : 0u);
        };
        // k values or more reach `lo`, fewer reach `hi`
        uint32_t lo = bound, hi = top_key + 1;
        bool few_enough = false;
        while (hi - lo > 1 && !few_enough) {
            const uint32_t mid = lo + (hi - lo) / 2;
            uint32_t count = 0;
            for (int c = threadIdx.x; c < pieces; c += ST_NT) {
                float v[PER];
                unpack<E>(piece(c), v);
#pragma unroll
                for (int i = 0; i < PER; ++i) count += key_of(v[i]) >= mid;
            }
            count = sum(count);
            if (count >= (uint32_t)f.k) lo = mid, few_enough = count <= (uint32_t)ST_NT;
            else hi = mid;
        }
        if (threadIdx.x == 0) s.few.n[0] = 0;
        __syncthreads();
        n = gather(few_enough ? lo : lo + 1);
        if (!few_enough) {   // and of those equal to the k-th, the first ids
            for (int base = 0; base < pieces && n < (uint32_t)f.k; base += ST_NT) {
                const int c = base + threadIdx.x;
                uint32_t mask = 0;
                if (c < pieces) {
                    float v[PER];
                    unpack<E>(piece(c), v);
#pragma unroll
                    for (int i = 0; i < PER; ++i) mask |= (uint32_t)(key_of(v[i]) == lo) << i;
                }
                uint32_t up = __popc(mask);
                const uint32_t mine = up;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += v;
                }
                turn ^= 1;
                if (lane == 31) s.counts[turn][warp] = up;
                __syncthreads();
                const uint32_t of_warp = lane < ST_NT / 32 ? s.counts[turn][lane] : 0u;
                uint32_t at = n + __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0u) + up - mine;
                for (; mask && at < (uint32_t)f.k; mask &= mask - 1, ++at) s.lists[at] = Few<ST_NT>::entry(value_of(lo), c * PER - skip + __ffs(mask) - 1);
                n = min((uint32_t)f.k, n + __reduce_add_sync(0xffffffffu, of_warp));
            }
            __syncthreads();
        }
    }
    Few<ST_NT> few = {s.few, s.lists, lane, warp, 32, 0};
    uint64_t kept = 0;
    if (few.begin(n)) few.answer(f, r, s.lists, n, 0, 0, 0.0, true, true, true, kept, a.ids + row, a.logp + row);
}
template <class E>
int sample_top_launch(const SampleArgs& a, cudaStream_t st) {
    AB_CHECK_ARG(a.rows <= INT32_MAX, "sampling: too many rows");
    // some 1.4 k values reach the bound where k is half the threads
    if (a.k_all <= 256) sample_top_kernel<E, 512><<<(unsigned)a.rows, 512, 0, st>>>(a);
    else sample_top_kernel<E, 1024><<<(unsigned)a.rows, 1024, 0, st>>>(a);
    AB_CUDA(cudaGetLastError());
    return OK;
}

template <class E>
int sample_keys_launch(SampleArgs a, cudaStream_t st) {
    static PerDeviceOnce once;
    const DeviceProps* dev;
    const auto kernel = sample_keys_kernel<E>;
    const int err = once.run(&dev, [&](const DeviceProps&) -> int {
        return check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(KeyShared)), "cudaFuncSetAttribute(sampling)");
    });
    if (err != OK) return err;
    AB_CHECK_ARG(a.rows <= INT32_MAX, "sampling: too many rows");
    a.ahead = dev->n_sm;
    kernel<<<(unsigned)a.rows, SK_NT, sizeof(KeyShared), st>>>(a);
    AB_CUDA(cudaGetLastError());
    return OK;
}

template <class E>
int sample_launch(SampleArgs a, cudaStream_t st) {
    constexpr int PER = 16 / sizeof(E), NT = 1024;
    static PerDeviceOnce once;
    static int fit[AB_MAX_DEVICES][4];   // clusters of 1, 2, 4 and 8 blocks that a device holds at a time
    const DeviceProps* dev;
    const auto kernel = sample_filtered_kernel<E, NT>;
    const int head = (int)sizeof(SampleShared<NT>);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    auto configure = [&](int64_t rows, int blocks, size_t smem) {
        cfg.gridDim = dim3((unsigned)(rows * blocks));
        cfg.blockDim = dim3(NT);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = blocks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    };
    const int err = once.run(&dev, [&](const DeviceProps& d) -> int {
        AB_CHECK_ARG(d.smem_optin >= (size_t)head + SP_ROW_BYTES, "sampling: %zu bytes of shared memory per block are too few", d.smem_optin);
        AB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, head + SP_ROW_BYTES));
        for (int i = 0; 1 << i <= SP_MAX_BLOCKS; ++i) {
            configure(1, 1 << i, (size_t)head + SP_ROW_BYTES);
            AB_CUDA(cudaOccupancyMaxActiveClusters(&fit[&d - once.props][i], kernel, &cfg));
        }
        return OK;
    });
    if (err != OK) return err;
    const int pieces = (a.V + 2 * PER - 2) / PER;   // wherever the row starts
    int lg = 0;
    while ((pieces + (1 << lg) - 1) / (1 << lg) * 16 > SP_ROW_BYTES) ++lg;
    AB_CHECK_ARG(1 << lg <= SP_MAX_BLOCKS, "sampling: a vocabulary of %d is too large", a.V);
    // More blocks to a row while all rows run at once, a piece or more to each thread. (fp32 65536, top-p: 1 row in eight blocks 48 us, in
    // two 62. But 16 rows in eight blocks, of which 128 SMs hold fewer than 16 clusters at a time, take two turns: under top-k 50 24.8 us,
    // in four 12.1.)
    while (1 << lg < SP_MAX_BLOCKS && a.rows <= fit[dev - once.props][lg + 1] && pieces > 1024 << lg) ++lg;
    const int blocks = 1 << lg;
    AB_CHECK_ARG(a.rows <= INT32_MAX / blocks, "sampling: too many rows");
    a.share = (pieces + blocks - 1) / blocks;
    configure(a.rows, blocks, (size_t)head + (size_t)a.share * 16);
    AB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    return OK;
}

}  // namespace

int sample_filtered(int dtype, int64_t rows, int V, const void* logits, int64_t stride, const float* u, const ab_sampling& p, int64_t* ids, float* logp, cudaStream_t st) {
    const SampleArgs a = {logits, u, p.temperature, p.top_p, p.min_p, p.top_k, p.temperature_all, p.top_p_all, p.min_p_all, p.top_k_all, V, rows, stride, ids, logp, 0, 0};
    // 16-bit rows of up to 65536: counters. Streamed instead where more rows than SMs have the same top-k of up to 256: 512 x 65536 fp16
    // with k of 50 41.8 us against 49.0, 256 54.1 against 63.1, but 400 81.0 against 72.3; 512 x 32003 27.5 against 37.5, 39.8 against
    // 50.3, 70.5 against 58.0; 512 x 5003 19.0 against 29.0, 31.6 against 39.3, 58.0 against 45.4. With 148 rows of k 50 19.1 against 16.0,
    // 14.5 against 12.9, 10.6 and 10.6; with one 14.7 against 12.9, 10.6 and 10.6, 9.3 against 8.6.
    const bool keys = V <= SK_BINS && dtype != AB_DT_F32, streams = !p.top_k && p.top_k_all > 0 && p.top_k_all <= ST_MOST_K && p.top_k_all < V;
    if (streams && !(keys && (rows <= current_sm_count() || p.top_k_all > 256)))
        return dtype == AB_DT_F16 ? sample_top_launch<__half>(a, st) : dtype == AB_DT_BF16 ? sample_top_launch<__nv_bfloat16>(a, st) : sample_top_launch<float>(a, st);
    if (keys) return dtype == AB_DT_F16 ? sample_keys_launch<__half>(a, st) : sample_keys_launch<__nv_bfloat16>(a, st);
    return dtype == AB_DT_F16 ? sample_launch<__half>(a, st) : dtype == AB_DT_BF16 ? sample_launch<__nv_bfloat16>(a, st) : sample_launch<float>(a, st);
}

}  // namespace ab
