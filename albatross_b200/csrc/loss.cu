// Log-probabilities of ids under rows of logits, the losses built on them, and their gradients by the logits.
//
// logp = x[id] - m - log(sum exp(x - m)) with m the row's maximum; d logp / dx = onehot(id) - exp(x - m) / sum.
#include <algorithm>
#include <type_traits>

#include "train.cuh"

namespace ab {

namespace {

constexpr int LT = 256;

struct RowTask {
    ab_logit_rows t;
    int policy;                  // 1: the row's loss and its derivative by logp too
    ab_policy p;
    double* logp;                // or null
    double *row_loss, *slope;    // the rows' losses and, or null, their derivatives by logp
    float *logp32, *stats;       // or null
    void* dlogits;               // null: no gradient in this pass
    const double* inv_denom;     // of the gradient in this pass
    float scale;
};

__device__ __forceinline__ bool counts(const ab_logit_rows& t, int64_t r) { return !t.mask || t.mask[r]; }

__device__ __forceinline__ int row_id(const ab_logit_rows& t, int64_t r) {
    const int64_t id = t.ids[r];
    if ((uint64_t)id < (uint64_t)t.vocab) return (int)id;
    if (threadIdx.x == 0) atomicOr(&g_device_status, DEV_BAD_TOKEN);
    return id < 0 ? 0 : t.vocab - 1;
}

struct PolicyRow {
    float A, old, ref;
};
__device__ __forceinline__ PolicyRow policy_load(const ab_policy& p, int64_t r) {
    return {p.advantages[r], p.old_logp ? p.old_logp[r] : 0.f, p.ref_logp ? p.ref_logp[r] : 0.f};
}
// What a row's loss and its derivative by the log-probability are made of, in 64 bits and the same whichever way the gradient is made: a ratio or the
// penalty's exponential may be infinite in 32 bits beside a factor that makes them small or nothing, and 1 - exp(gap) is small where the reference is
// near. With logp = rel - log(S) the logarithm is not needed: ratio = exp(rel - old) / S, exp(gap) = exp(ref - rel) S. A factor of 0 counts for more
// than an infinite ratio: the ratio's exponential is held finite (exp(709) is; a NaN stays one), and without a weight the reference is not looked at.
struct PolicyTerms {
    double least, slope, e;      // min(ratio A, clipped A); the derivative by logp; exp(gap), or 1
    __device__ __forceinline__ double loss(const ab_policy& p, const PolicyRow& q, double logp) const {
        return -least + (p.ref_logp && p.kl != 0.f ? (double)p.kl * (e - ((double)q.ref - logp) - 1.0) : 0.0);
    }
};
// By a whole warp: its even lanes take the ratio's exponential, its odd ones the penalty's. All of a row's other warps wait for the slope. (old: the
// ratio is not 1; kl 0: no reference)
__device__ __forceinline__ PolicyTerms policy_terms(bool old, float old_logp, float A, float low, float high, float kl, float ref_logp, double rel, float S) {
    const bool odd = threadIdx.x & 1;
    const double x = odd ? (kl != 0.f ? (double)ref_logp - rel : 0.0) : old ? rel - (double)old_logp : 0.0;
    const double f = exp(x > 709.0 && !odd ? 709.0 : x);
    const float near = 1.f / S;
    const double inv = fma((double)near, fma(-(double)S, (double)near, 1.0), (double)near);   // 1 / S to 2^-46
    const double ratio = old ? __shfl_sync(0xffffffffu, f, 0) * inv : 1.0, most = 1.0 + (double)high, fewest = 1.0 - (double)low;
    const bool cut = (A > 0.f && ratio > most) || (A < 0.f && ratio < fewest);
    const double plain = ratio * (double)A;
    PolicyTerms t;
    t.e = kl != 0.f ? __shfl_sync(0xffffffffu, f, 1) * (double)S : 1.0;
    t.least = cut ? (A > 0.f ? most : fewest) * (double)A : plain;
    t.slope = (cut ? 0.0 : -plain) + (kl != 0.f ? (double)kl * (1.0 - t.e) : 0.0);
    return t;
}
__device__ __forceinline__ float policy_kl(const ab_policy& p) { return p.ref_logp ? p.kl : 0.f; }
__device__ __forceinline__ PolicyTerms policy_terms(const ab_policy& p, const PolicyRow& q, double rel, float S) {
    return policy_terms(p.old_logp != nullptr, q.old, q.A, p.clip_low, p.clip_high, policy_kl(p), q.ref, rel, S);
}
// The same where every register counts: inlined, it made the rows' exponentials spill (4096 x 9001 fp16 rows with gradient 90 us, called 85; 4096 x
// 32003 in the ring the other way round, 158 and 165).
__device__ __noinline__ PolicyTerms policy_terms_call(bool old, float old_logp, float A, float low, float high, float kl, float ref_logp, double rel, float S) {
    return policy_terms(old, old_logp, A, low, high, kl, ref_logp, rel, S);
}
__device__ __forceinline__ PolicyTerms policy_terms_apart(const ab_policy& p, const PolicyRow& q, double rel, float S) {
    return policy_terms_call(p.old_logp != nullptr, q.old, q.A, p.clip_low, p.clip_high, policy_kl(p), q.ref, rel, S);
}

// ---- a row in registers --------------------------------------------------------------------------------------------
// A row is taken in pieces of 16 bytes on 16-byte addresses, whatever address it starts on: the first and the last piece may hold
// values of its neighbours, which count as -inf and are not written.
template <class E>
struct Pieces {
    static constexpr int N = 16 / sizeof(E);
    const E* x;        // the first piece's address
    int lead, n, V;    // values of the first piece in front of the row; pieces; values of the row
    Extent in;         // the rows' whole array
    __device__ __forceinline__ Pieces(const E* row, int V_, const Extent& in_) : V(V_), in(in_) {
        lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
        x = row - lead;
        n = (V + lead + N - 1) / N;
    }
    // pieces i0 .. i1 - 1 hold values of the row alone
    __device__ __forceinline__ bool all_whole(int i0, int i1) const { return i0 * N >= lead && i1 * N <= V + lead; }
    template <bool FULL>
    __device__ __forceinline__ uint4 get(int i) const {
        if (FULL) return piece(i);
        return load(i);
    }
    __device__ __forceinline__ bool whole(int i) const { return i * N >= lead && (i + 1) * N <= V + lead; }
    __device__ __forceinline__ uint4 load(int i) const {
        if (i >= n) return none();
        if (whole(i)) return piece(i);
        uint4 u = none();
        E* e = reinterpret_cast<E*>(&u);
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (i * N + c >= lead && i * N + c < V + lead && in.holds(x + i * N + c)) e[c] = x[i * N + c];
        return u;
    }
    __device__ __forceinline__ uint4 piece(int i) const {
        const uint4* p = reinterpret_cast<const uint4*>(x) + i;
        return in.holds(p) ? __ldcs(p) : none();
    }
    __device__ __forceinline__ float value(int id) const { return in.holds(x + lead + id) ? to_f(x[lead + id]) : 0.f; }
    static __device__ __forceinline__ uint4 none() {   // -inf throughout
        const uint32_t w = sizeof(E) == 4 ? 0xff800000u : std::is_same<E, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        return make_uint4(w, w, w, w);
    }
};
// the larger values of two pieces, place by place (a NaN gives way: it is left to the sums), and the largest of one
template <class E>
__device__ __forceinline__ uint4 piece_max(uint4 a, const uint4& b) {
    uint32_t *x = &a.x;
    const uint32_t* y = &b.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<E, float>::value) x[i] = __float_as_uint(fmaxf(__uint_as_float(x[i]), __uint_as_float(y[i])));
        else if constexpr (std::is_same<E, __half>::value) asm("max.f16x2 %0, %0, %1;" : "+r"(x[i]) : "r"(y[i]));
        else asm("max.bf16x2 %0, %0, %1;" : "+r"(x[i]) : "r"(y[i]));
    }
    return a;
}
template <class E>
__device__ __forceinline__ float piece_top(const uint4& u) {
    float f[Pieces<E>::N];
    unpack<E>(u, f);
    float m = f[0];
#pragma unroll
    for (int c = 1; c < Pieces<E>::N; ++c) m = fmaxf(m, f[c]);
    return m;
}
// What exponentials are taken relative to: exp(x - m) = 2^(x log2(e) - c) with c = m log2(e) rounded, one multiply-add and one ex2.approx (good to
// 2^-22). Joining parts takes the difference of two c, so that the rounding of c cancels. The constant's own rounding, 2^-25.7 of x, is left out of
// the gradient's exponentials only; beyond |m| = 64 it would count, as would c's, and at the type's ends (rows of the lowest value throughout, which
// some programs use for a mask) the product overflows: there the difference comes first.
constexpr float LOG2E = 1.4426950408889634f, LOG2E_LOW = 1.925963033500e-8f;   // log2(e), and what its 24 bits leave of it
struct Ref {
    float m, c;
    bool huge;
    __device__ __forceinline__ Ref(float top) : m(top == -INFINITY ? 0.f : top), c(m * LOG2E), huge(fabsf(m) > 64.f) {}   // (nothing above -inf: sums of 0 or NaN)
};
__device__ __forceinline__ float ex2(float x) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    return e;
}
template <int N>
__device__ __forceinline__ void exp_from(float* f, const Ref& r) {
    if (r.huge) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = ex2((f[i] - r.m) * LOG2E);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = ex2(fmaf(f[i], LOG2E, -r.c));
    }
}
// The same for sums, with the constant in two parts: one part alone is off by 1.3e-8 of it, which all of a row's exponentials share, so that
// log-probabilities of -10 were off by 1e-7 to one side and mean losses with them.
template <int N>
__device__ __forceinline__ void exp_to_add(float* f, const Ref& r) {
    if (r.huge) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] -= r.m, f[i] = ex2(fmaf(f[i], LOG2E_LOW, f[i] * LOG2E));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = ex2(fmaf(f[i], LOG2E_LOW, fmaf(f[i], LOG2E, -r.c)));
    }
}
__device__ __forceinline__ float exp_from(float x, const Ref& r) {
    exp_from<1>(&x, r);
    return x;
}
// 2^x for factors of whole sums, by the series of exp((x - n) log(2)) up to the seventh power, n the nearest integer: within 2^-23 and to neither
// side. (ex2.approx is 4e-8 too small on average; a sum goes through two or three factors on its way, so that log-probabilities over 65536 values
// were 1.1e-7 too large, and are 5e-8 now, for 1.5% of the time of 4096 rows.)
__device__ __forceinline__ float ex2_factor(float x) {
    if (!(fabsf(x) < 126.f)) return ex2(x);
    const float n = rintf(x), y = (x - n) * 0.69314718f;
    float p = 1.f / 5040.f;
    p = fmaf(p, y, 1.f / 720.f);
    p = fmaf(p, y, 1.f / 120.f);
    p = fmaf(p, y, 1.f / 24.f);
    p = fmaf(p, y, 1.f / 6.f);
    p = fmaf(p, y, 0.5f);
    p = fmaf(p, y, 1.f);
    p = fmaf(p, y, 1.f);
    return p * __int_as_float((int)(n + 127.f) << 23);
}
// 2^(difference of two references): what a sum relative to the first becomes relative to the second
__device__ __forceinline__ float rebase(const Ref& from, const Ref& to) {
    float d = from.c - to.c;
    if (from.huge && to.huge) {
        const float m = from.m - to.m;
        d = fmaf(m, LOG2E_LOW, m * LOG2E);
    } else if (from.huge || to.huge) {
        const float m = from.huge ? from.m : to.m, x = fmaf(m, LOG2E_LOW, fmaf(m, LOG2E, -(from.huge ? to.c : from.c)));
        d = from.huge ? x : -x;
    }
    return ex2_factor(d);
}
// Writes p times a piece's exponentials to the row `dx`, which starts `lead` values into a piece of 16 bytes as the row of logits does (aligned), or
// anywhere. FULL: the piece holds values of the row alone, and dx is aligned.
template <class E, bool FULL>
__device__ __forceinline__ void write_piece(const Pieces<E>& row, const float* e, int i, E* dx, bool aligned, float p, const Extent& grads) {
    constexpr int N = Pieces<E>::N;
    if (!FULL && i >= row.n) return;
    float f[N];
#pragma unroll
    for (int c = 0; c < N; ++c) f[c] = e[c] * p;
    const int first = i * N - row.lead;
    const uint4 out = pack<E>(f);
    if (FULL || (aligned && row.whole(i))) {
        uint4* to = reinterpret_cast<uint4*>(dx - row.lead) + i;
        if (grads.holds(to)) __stcs(to, out);
    } else {
        const E* o = reinterpret_cast<const E*>(&out);
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (first + c >= 0 && first + c < row.V && grads.holds(dx + first + c)) dx[first + c] = o[c];
    }
}
template <class E>
__device__ __forceinline__ void write_zeros(E* dx, int V, int at, int step, const Extent& grads) {   // this thread's share: pieces at, at + step, ...
    const Pieces<E> row(dx, V, grads);
    for (int i = at; i < row.n; i += step) {
        const int first = i * Pieces<E>::N - row.lead;
        if (row.whole(i)) {
            if (grads.holds(reinterpret_cast<uint4*>(dx + first))) __stcs(reinterpret_cast<uint4*>(dx + first), make_uint4(0, 0, 0, 0));
        } else {
            for (int c = max(first, 0); c < min(first + Pieces<E>::N, V); ++c)
                if (grads.holds(dx + c)) dx[c] = from_f<E>(0.f);
        }
    }
}

template <class E>
__device__ __forceinline__ Extent logits_extent(const ab_logit_rows& t) { return rows_extent(t.logits, t.rows, t.stride, t.vocab, sizeof(E)); }
template <class E>
__device__ __forceinline__ Extent grads_extent(const ab_logit_rows& t, const void* dlogits) { return rows_extent(dlogits, t.rows, t.vocab, t.vocab, sizeof(E)); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_blocks() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

constexpr int LW = LT / 32, MAX_CLUSTER = 8;

__device__ __forceinline__ float warp_top(float v) {   // warp_max in one instruction
    asm("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
    return v;
}

// A row's maximum and sum, in every lane, from the warps' parts that the lanes hold (one of no values has sum 0 or NaN), in one order.
struct RowSum {
    float M;
    Ref ref;
    float S;
    __device__ __forceinline__ RowSum(const float2& a, const float2& b) : M(warp_top(fmaxf(a.x, b.x))), ref(M) {
        S = warp_sum(a.y * (a.x == -INFINITY ? 1.f : rebase(Ref(a.x), ref)) + b.y * (b.x == -INFINITY ? 1.f : rebase(Ref(b.x), ref)));
        if (M == -INFINITY) S = NAN;                       // no probabilities to speak of
    }
};
// a value relative to the reference
__device__ __forceinline__ double relative(float at, const Ref& ref) {
    return ref.huge ? (double)at - (double)ref.m : ((double)at * 1.4426950408889634074 - (double)ref.c) * 0.6931471805599453094;
}

// rows that count, up to all of them, as this thread's share of a block of LT
__device__ __forceinline__ int count_rows(const uint8_t* mask, int64_t rows) {
    if (!mask) return threadIdx.x == 0 ? (int)rows : 0;
    const int lead = (int)min((int64_t)((16 - (reinterpret_cast<uintptr_t>(mask) & 15)) & 15), rows), pieces = (int)((rows - lead) / 16);
    int n = 0;
    for (int i = threadIdx.x; i < pieces; i += LT) {
        const uint4* p = reinterpret_cast<const uint4*>(mask + lead) + i;
        const uint4 u = Extent(mask, rows).holds(p) ? *p : make_uint4(0, 0, 0, 0);   // bytes of 0 and 1
        n = __dp4a(u.x, 0x01010101u, __dp4a(u.y, 0x01010101u, __dp4a(u.z, 0x01010101u, __dp4a(u.w, 0x01010101u, (unsigned)n))));
    }
    if ((int)threadIdx.x < lead) n += mask[threadIdx.x];
    const int64_t tail = lead + (int64_t)pieces * 16 + threadIdx.x;
    if (threadIdx.x < 16 && tail < rows) n += mask[tail];
    return n;
}

// One row per cluster of blocks, a run of pieces per block; a thread keeps the exponentials of EPT values in registers between the sums and the
// gradient, so that the logits are read once and each exponential is taken once (rows longer than MAX_CLUSTER * LT * EPT values are read twice).
template <class E, int EPT>
__global__ void __launch_bounds__(LT, 4) logit_rows_kernel(const __grid_constant__ RowTask k) {
    constexpr int N = Pieces<E>::N, NV = EPT / N;
    __shared__ float2 part[MAX_CLUSTER * LW];   // maximum and sum of every warp of the cluster
    __shared__ int s_count[LW];
    __shared__ float4 s_join;
    const uint32_t rank = cluster_rank(), nb = cluster_blocks();
    const int64_t r = blockIdx.x / nb;
    const int V = k.t.vocab, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    E* dx = k.dlogits ? static_cast<E*>(k.dlogits) + r * V : nullptr;
    const Extent grads = grads_extent<E>(k.t, k.dlogits);
    pdl_launch_dependents();
    if (!AB_BC(r < k.t.rows)) return;
    if (!counts(k.t, r)) {
        if (tid == 0 && rank == 0) {
            if (k.logp) k.logp[r] = 0.0;
            if (k.logp32) k.logp32[r] = 0.f;
            if (k.row_loss) k.row_loss[r] = 0.0;
            if (k.slope) k.slope[r] = 0.0;
            if (k.stats) k.stats[2 * r] = k.stats[2 * r + 1] = 0.f;
        }
        if (dx) write_zeros(dx, V, (int)rank * LT + tid, (int)nb * LT, grads);
        return;
    }
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (the blocks of a row all come here: its mask is theirs)
    const Pieces<E> row(static_cast<const E*>(k.t.logits) + r * k.t.stride, V, logits_extent<E>(k.t));
    const int step = (int)nb * LT * NV, at0 = (int)rank * LT * NV;
    const bool aligned = dx && (reinterpret_cast<uintptr_t>(dx) & 15) == row.lead * sizeof(E);
    const bool once = row.n <= step, full = once && row.all_whole(at0, at0 + LT * NV) && (aligned || !dx);
    float e[EPT], m = -INFINITY, s = 0.f, at = 0.f;
    int id = 0;
    PolicyRow pr = {};
    auto sums = [&](auto whole, int base) {
        uint4 u[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) u[j] = row.template get<decltype(whole)::value>(base + at0 + j * LT + tid);
        if (base == 0) {
            id = row_id(k.t, r);
            at = row.value(id);
            if (k.policy) pr = policy_load(k.p, r);
        }
        uint4 top4 = u[0];
#pragma unroll
        for (int j = 1; j < NV; ++j) top4 = piece_max<E>(top4, u[j]);
        const float top = warp_top(fmaxf(m, piece_top<E>(top4)));
        const Ref ref(top);
        if (m != top) s *= m == -INFINITY ? 1.f : rebase(Ref(m), ref), m = top;   // (m -inf: s is 0 or NaN, and stays so)
        float sum[4] = {s, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) unpack<E>(u[j], e + j * N);
        exp_to_add<EPT>(e, ref);
#pragma unroll
        for (int c = 0; c < EPT; ++c) sum[c & 3] += e[c];
        s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    if (full) sums(std::true_type(), 0);
    else
        for (int base = 0; base < row.n; base += step) sums(std::false_type(), base);
    s = warp_sum(s);
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every block of the cluster has started: its shared memory may be written
    if (lane < (int)nb) {                                  // to every block of the cluster
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(&part[rank * LW + warp])), "r"(lane));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(m), "f"(s) : "memory");
    }
    const bool counting = k.policy && dx && !k.inv_denom;  // every block counts the rows that count, for the loss's denominator
    if (counting) {
        const int n = __reduce_add_sync(0xffffffffu, count_rows(k.t.mask, k.t.rows));
        if (lane == 0) s_count[warp] = n;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) {
        // one warp joins the parts, in one order
        float2 a = make_float2(-INFINITY, 0.f), b = a;
        const int n_parts = (int)nb * LW;
        if (lane < n_parts) a = part[lane];
        if (lane + 32 < n_parts) b = part[lane + 32];
        const RowSum t(a, b);
        const double rel = relative(at, t.ref);
        PolicyTerms terms = {};
        if (dx) {
            int n = 0;
            if (counting)
                for (int i = 0; i < LW; ++i) n += s_count[i];
            terms = policy_terms_apart(k.p, pr, rel, t.S);
            const float g = (float)(terms.slope * ((counting ? 1.0 / (double)max(n, 1) : *k.inv_denom) * (double)k.scale));
            if (lane == 0) s_join = make_float4(t.M, -g / t.S, g, 0.f);
            __syncwarp();
            asm volatile("bar.arrive 1, %0;" ::"n"(LT) : "memory");
        }
        if (k.policy && !dx && rank == 0) terms = policy_terms_apart(k.p, pr, rel, t.S);
        if (lane == 0 && rank == 0) {                      // (while the other warps write)
            const double logp = rel - log((double)t.S);
            if (k.logp) k.logp[r] = logp;
            if (k.logp32) k.logp32[r] = (float)logp;
            if (k.stats) {
                k.stats[2 * r] = t.M;
                k.stats[2 * r + 1] = 1.f / t.S;
            }
            if (k.policy) {
                k.row_loss[r] = terms.loss(k.p, pr, logp);
                if (k.slope) k.slope[r] = terms.slope;
            }
        }
    }
    if (!dx) return;
    if (warp != 0) asm volatile("bar.sync 1, %0;" ::"n"(LT) : "memory");
    else __syncwarp();
    const float4 join = s_join;
    const float M = join.x, p = join.y, g = join.z;
    const Ref ref(M);
    const float mine = p * (m == -INFINITY ? 1.f : rebase(Ref(m), ref));   // the exponentials are relative to the warp's maximum
    if (full) {
#pragma unroll
        for (int j = 0; j < NV; ++j) write_piece<E, true>(row, e + j * N, at0 + j * LT + tid, dx, aligned, mine, grads);
    } else if (once) {
#pragma unroll
        for (int j = 0; j < NV; ++j) write_piece<E, false>(row, e + j * N, at0 + j * LT + tid, dx, aligned, mine, grads);
    } else {
        for (int i = at0; i < row.n; i += step)
            for (int j = 0; j < NV; ++j) {
                unpack<E>(row.load(i + j * LT + tid), e);
                exp_from<N>(e, ref);
                write_piece<E, false>(row, e, i + j * LT + tid, dx, aligned, p, grads);
            }
    }
    // the id's own value, by the thread that wrote its piece
    const int own = (id + row.lead) / N - at0;
    if (own >= 0 && own % step < LT * NV && own % LT == tid && grads.holds(dx + id)) dx[id] = from_f<E>(fmaf(p, exp_from(at, ref), g));
}

// ---- long rows, at least one per SM ----------------------------------------------------------------------------------
// One block per SM takes row after row: a warp asks for a row's chunks with bulk copies into a ring, ahead of the warps that add them up and then go
// through the ring once more for the gradient; as they hand chunks back the next row's come in, so that copies are under way through the sums, the
// join and the gradient alike. Which row comes next is asked of the hardware (cluster launch control: the grid has a block per row, and a running
// block takes the place of one that has not started), because masked rows cost little and would unbalance fixed shares. What a row needs besides its
// logits (id, policy) travels the same way ahead of it; a row's own log-probability and loss, in 64 bits, are the business of another warp. 4096 x
// 65536 fp16 rows, the policy loss with its gradient (85 % of the rows count, the others' logits are not read): 243 us for 0.99 GB, 4.1 TB/s, 63 % of
// the copy rate. 21 instructions a value at 2.2 a cycle; without a gradient 11 at 2.4, 111 us (20 to 28 working warps, smaller or larger chunks and a
// chunk kept ahead in registers: slower by 8 to 60 %).
constexpr int RING_WARPS = 16, RING_THREADS = (RING_WARPS + 2) * 32, RING_CHUNK = 32768, RING_SLOTS = 7, RING_ROWS = 4;   // working warps; chunks, rows under way
struct RingRow {
    int64_t r;          // -1: no more
    int on, id;
    float at;
    PolicyRow pr;
    float g;            // from the finishing warp, where a gradient is made: its coefficient
    float2 part[RING_WARPS];   // the working warps' maxima and sums
};
struct RingShared {
    uint4 cancel;
    uint64_t full[RING_SLOTS], vacant[RING_SLOTS], row_full[RING_ROWS], row_summed[RING_ROWS], row_sloped[RING_ROWS], row_vacant[RING_ROWS], cancelled;
    RingRow row[RING_ROWS];
    int count[RING_WARPS + 2], failed;
    uint32_t nobody;
};

template <class E>
__global__ void __launch_bounds__(RING_THREADS, 1) logit_ring_kernel(const __grid_constant__ RowTask k) {
    constexpr int N = Pieces<E>::N, PER = RING_CHUNK / 16 / (RING_WARPS * 32);   // a thread's pieces of a chunk
    extern __shared__ __align__(128) unsigned char ring[];            // RING_SLOTS chunks
    __shared__ RingShared sh;
    const int V = k.t.vocab, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < RING_SLOTS; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.vacant[i], RING_WARPS);
        for (int i = 0; i < RING_ROWS; ++i) {
            mbar_init(&sh.row_full[i], 1), mbar_init(&sh.row_summed[i], RING_WARPS);
            mbar_init(&sh.row_sloped[i], 1), mbar_init(&sh.row_vacant[i], RING_WARPS + 1);
        }
        mbar_init(&sh.cancelled, 1);
        fence_mbar_init();
        sh.failed = 0;
    }
    const bool counting = k.policy && k.dlogits && !k.inv_denom;
    if (counting) {
        int n = 0;
        for (int64_t i = tid; i < k.t.rows; i += RING_THREADS) n += counts(k.t, i) ? 1 : 0;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) sh.count[warp] = n;
    }
    __syncthreads();
    pdl_launch_dependents();
    // after the first wait that runs out nobody waits any more
    auto wait_for = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile int*>(&sh.failed)) return false;
        if (mbar_wait_bounded(bar, parity, 1u << 18)) return true;
        *reinterpret_cast<volatile int*>(&sh.failed) = 1;
        atomicOr(&g_device_status, DEV_WAIT_HEAD);
        return false;
    };
    const E* logits = static_cast<const E*>(k.t.logits);
    const Extent in = logits_extent<E>(k.t), grads = grads_extent<E>(k.t, k.dlogits);
    // the pieces of a row that are copied: those that hold its values alone
    auto span = [&](const Pieces<E>& row, int& first, int& end) {
        first = row.lead ? 1 : 0;
        end = (V + row.lead) / N;
    };
    constexpr int CP = RING_CHUNK / 16;   // pieces of a chunk

    if (warp == RING_WARPS) {
        if (lane == 0) {
            int64_t r = blockIdx.x;
            int c_issued = 0, asked = 0, answered = 0;
            bool ok = true;
            for (int n = 0; ok; ++n) {
                RingRow& q = sh.row[n % RING_ROWS];
                if (n >= RING_ROWS && !wait_for(&sh.row_vacant[n % RING_ROWS], (uint32_t)(n / RING_ROWS - 1) & 1u)) break;
                if (r >= 0) {
                    // ask for the row after this one
                    fence_proxy_async();
                    ++asked;
                    mbar_expect_tx(&sh.cancelled, 16);
                    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(&sh.cancel)),
                                 "r"(smem_u32(&sh.cancelled)) : "memory");
                }
                q.r = r;
                if (r >= 0) {
                    q.on = counts(k.t, r);
                    if (q.on) {
                        const Pieces<E> row(logits + r * k.t.stride, V, in);
                        int first, end;
                        span(row, first, end);
                        const int chunks = (end - first + CP - 1) / CP, rounds = chunks > RING_SLOTS && k.dlogits ? 2 : 1;
                        bool published = false;
                        for (int round = 0; round < rounds && ok; ++round)
                            for (int c = 0; c < chunks && ok; ++c, ++c_issued) {
                                const int slot = c_issued % RING_SLOTS, p0 = first + c * CP, np = min(CP, end - p0);
                                if (c_issued >= RING_SLOTS) ok = wait_for(&sh.vacant[slot], (uint32_t)(c_issued / RING_SLOTS - 1) & 1u);
                                if (!ok) break;
                                const uint4* from = reinterpret_cast<const uint4*>(row.x) + p0;
                                if (in.holds(from, np) && AB_BC(slot >= 0 && np > 0 && slot * RING_CHUNK + np * 16 <= RING_SLOTS * RING_CHUNK && np * 16 <= RING_CHUNK)) {
                                    mbar_expect_tx(&sh.full[slot], np * 16);
                                    bulk_g2s(ring + (size_t)slot * RING_CHUNK, from, np * 16, &sh.full[slot]);
                                } else {
                                    mbar_arrive(&sh.full[slot]);
                                }
                                if (!published) {                        // the rest of what the row needs, while its first chunk travels
                                    published = true;
                                    const int64_t id = k.t.ids[r];
                                    q.id = (uint64_t)id < (uint64_t)V ? (int)id : (atomicOr(&g_device_status, DEV_BAD_TOKEN), id < 0 ? 0 : V - 1);
                                    q.at = row.value(q.id);
                                    if (k.policy) q.pr = policy_load(k.p, r);
                                    mbar_arrive(&sh.row_full[n % RING_ROWS]);
                                }
                            }
                    } else {
                        mbar_arrive(&sh.row_full[n % RING_ROWS]);
                    }
                    if (!ok || !wait_for(&sh.cancelled, (uint32_t)n & 1u)) break;
                    ++answered;
                    uint32_t got, next;
                    asm volatile("{\n .reg .pred p;\n .reg .b128 h;\n ld.shared.b128 h, [%2];\n"
                                 " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
                                 " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n}"
                                 : "=r"(got), "=r"(next) : "r"(smem_u32(&sh.cancel)) : "memory");
                    r = got && AB_BC(next < k.t.rows) ? (int64_t)next : -1;
                } else {
                    mbar_arrive(&sh.row_full[n % RING_ROWS]);
                    break;
                }
            }
            // whatever became of the waits, all that was asked for lands before the block ends
            for (int c = max(0, c_issued - RING_SLOTS); c < c_issued; ++c) mbar_wait_bounded(&sh.full[c % RING_SLOTS], (uint32_t)(c / RING_SLOTS) & 1u, 1u << 18);
            if (answered < asked) mbar_wait_bounded(&sh.cancelled, (uint32_t)answered & 1u, 1u << 18);
        }
    } else if (warp == RING_WARPS + 1) {
        double inv_n = k.inv_denom ? *k.inv_denom : 1.0;
        if (counting) {
            int n = 0;
            for (int i = 0; i < RING_WARPS + 2; ++i) n += sh.count[i];
            inv_n = 1.0 / (double)max(n, 1);
        }
        inv_n *= (double)k.scale;
        for (int n = 0;; ++n) {
            RingRow& q = sh.row[n % RING_ROWS];
            if (!__all_sync(0xffffffffu, wait_for(&sh.row_full[n % RING_ROWS], (uint32_t)(n / RING_ROWS) & 1u)) || q.r < 0) break;
            if (!__all_sync(0xffffffffu, wait_for(&sh.row_summed[n % RING_ROWS], (uint32_t)(n / RING_ROWS) & 1u))) break;
            double logp = 0.0, loss = 0.0, slope = 0.0;
            float M = 0.f, inv_s = 0.f;
            if (q.on) {
                const float2 none = make_float2(-INFINITY, 0.f);
                const RowSum t(lane < RING_WARPS ? q.part[lane] : none, none);
                const double rel = relative(q.at, t.ref);
                if (k.policy) {
                    const PolicyTerms terms = policy_terms(k.p, q.pr, rel, t.S);
                    slope = terms.slope;
                    if (k.dlogits && lane == 0) {
                        q.g = (float)(slope * inv_n);
                        mbar_arrive(&sh.row_sloped[n % RING_ROWS]);
                    }
                    logp = rel - log((double)t.S);
                    loss = terms.loss(k.p, q.pr, logp);
                } else {
                    logp = rel - log((double)t.S);
                }
                M = t.M, inv_s = 1.f / t.S;
            } else if (k.dlogits && lane == 0) {
                mbar_arrive(&sh.row_sloped[n % RING_ROWS]);
            }
            if (lane == 0) {
                if (k.logp) k.logp[q.r] = logp;
                if (k.logp32) k.logp32[q.r] = (float)logp;
                if (k.stats) k.stats[2 * q.r] = M, k.stats[2 * q.r + 1] = inv_s;
                if (k.policy) k.row_loss[q.r] = loss;
                if (k.slope) k.slope[q.r] = slope;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.row_vacant[n % RING_ROWS]);
        }
    } else {
        int c_seen = 0;
        for (int n = 0;; ++n) {
            RingRow& q = sh.row[n % RING_ROWS];
            if (!__all_sync(0xffffffffu, wait_for(&sh.row_full[n % RING_ROWS], (uint32_t)(n / RING_ROWS) & 1u))) break;
            const int64_t r = q.r;
            if (r < 0) break;
            E* dx = k.dlogits ? static_cast<E*>(k.dlogits) + r * V : nullptr;
            if (!q.on) {
                if (dx) write_zeros(dx, V, tid, RING_WARPS * 32, grads);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.row_summed[n % RING_ROWS]), mbar_arrive(&sh.row_vacant[n % RING_ROWS]);
                continue;
            }
            const Pieces<E> row(logits + r * k.t.stride, V, in);
            int first, end;
            span(row, first, end);
            const int chunks = (end - first + CP - 1) / CP;
            const bool twice = chunks > RING_SLOTS && dx;
            // the two ends of a row that are not copied, by the first two threads
            const int edge = tid == 0 && first ? 0 : tid == 1 && end < row.n ? end : -1;
            uint4 eu = Pieces<E>::none();
            if (edge >= 0) eu = row.load(edge);
            float m = -INFINITY, s = 0.f;
            auto add = [&](const uint4* u, int np) {
                uint4 t4 = u[0];
                for (int j = 1; j < np; ++j) t4 = piece_max<E>(t4, u[j]);
                const float top = warp_top(fmaxf(m, piece_top<E>(t4)));
                const Ref ref(top);
                if (m != top) s *= m == -INFINITY ? 1.f : rebase(Ref(m), ref), m = top;
                float sum[4] = {s, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (j >= np) break;
                    float e[N];
                    unpack<E>(u[j], e);
                    exp_to_add<N>(e, ref);
#pragma unroll
                    for (int c = 0; c < N; ++c) sum[c & 3] += e[c];
                }
                s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            };
            if (warp == 0) add(&eu, 1);
            auto hand_back = [&](int slot, const uint4* u) {
                uint32_t used = 0;
#pragma unroll
                for (int j = 0; j < PER; ++j) used ^= u[j].x ^ u[j].w;
                loads_returned(used, &sh.nobody);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.vacant[slot]);
            };
            auto take = [&](int c, uint4* u) {   // chunk c of the row
                const int slot = c_seen % RING_SLOTS, np = end - first - c * CP;
                wait_for(&sh.full[slot], (uint32_t)(c_seen / RING_SLOTS) & 1u);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int i = j * RING_WARPS * 32 + tid;
                    u[j] = i < np ? *reinterpret_cast<const uint4*>(ring + (size_t)slot * RING_CHUNK + i * 16) : Pieces<E>::none();
                }
                ++c_seen;
                return slot;
            };
            const int c0 = c_seen;
            for (int c = 0; c < chunks; ++c) {
                uint4 u[PER];
                const int slot = take(c, u);
                add(u, PER);
                if (!dx || twice) hand_back(slot, u);
            }
            s = warp_sum(s);
            if (lane == 0) {
                q.part[warp] = make_float2(m, s);
                mbar_arrive(&sh.row_summed[n % RING_ROWS]);
            }
            if (dx) {
                wait_for(&sh.row_summed[n % RING_ROWS], (uint32_t)(n / RING_ROWS) & 1u);
                __syncwarp();
                const float2 none = make_float2(-INFINITY, 0.f);
                const RowSum t(lane < RING_WARPS ? q.part[lane] : none, none);
                const Ref ref = t.ref;
                const float S = t.S, at = q.at;
                const int id = q.id;
                const bool aligned = (reinterpret_cast<uintptr_t>(dx) & 15) == row.lead * sizeof(E);
                float g = 0.f, p = 0.f;
                auto slope = [&]() {   // taken by the finishing warp, beside the first exponentials
                    wait_for(&sh.row_sloped[n % RING_ROWS], (uint32_t)(n / RING_ROWS) & 1u);
                    __syncwarp();
                    g = q.g, p = -g / S;
                };
                if (chunks == 0) slope();
                if (!twice) c_seen = c0;
                for (int c = 0; c < chunks; ++c) {
                    uint4 u[PER];
                    const int slot = take(c, u);
                    hand_back(slot, u);
                    float e[PER][N];
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        unpack<E>(u[j], e[j]);
                        exp_from<N>(e[j], ref);
                    }
                    if (c == 0) slope();
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const int i = c * CP + j * RING_WARPS * 32 + tid;
                        if (i < end - first) {
                            if (aligned) write_piece<E, true>(row, e[j], first + i, dx, true, p, grads);
                            else write_piece<E, false>(row, e[j], first + i, dx, false, p, grads);
                        }
                    }
                }
                if (edge >= 0) {
                    float e[N];
                    unpack<E>(eu, e);
                    exp_from<N>(e, ref);
                    write_piece<E, false>(row, e, edge, dx, aligned, p, grads);
                }
                // the id's own value, by the thread that wrote its piece
                const int piece = (id + row.lead) / N;
                const bool mine = piece >= first && piece < end ? (piece - first) % (RING_WARPS * 32) == tid : piece == edge;
                if (mine && grads.holds(dx + id)) dx[id] = from_f<E>(fmaf(p, exp_from(at, ref), g));
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.row_vacant[n % RING_ROWS]);
        }
    }
}

// ---- short rows --------------------------------------------------------------------------------------------------------
// Up to 1024 values: a warp per row, which then needs no other warp. (4096 rows of 1000 fp16 values with gradients: a block per row takes 30 us.)
constexpr int SHORT_EPT = 32;
template <class E>
__global__ void __launch_bounds__(LT, 3) logit_short_kernel(const __grid_constant__ RowTask k) {
    constexpr int N = Pieces<E>::N, NV = SHORT_EPT / N;
    __shared__ int s_count[LW];
    const int V = k.t.vocab, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    double inv_n = 0.0;
    if (k.policy && k.dlogits) {
        if (k.inv_denom) {
            inv_n = *k.inv_denom;
        } else {                                   // every block counts the rows that count
            const int n = __reduce_add_sync(0xffffffffu, count_rows(k.t.mask, k.t.rows));
            if (lane == 0) s_count[warp] = n;
            __syncthreads();
            int all = 0;
            for (int i = 0; i < LW; ++i) all += s_count[i];
            inv_n = 1.0 / (double)max(all, 1);
        }
    }
    const int64_t r = (int64_t)blockIdx.x * LW + warp;
    if (r >= k.t.rows) return;
    E* dx = k.dlogits ? static_cast<E*>(k.dlogits) + r * V : nullptr;
    const Extent grads = grads_extent<E>(k.t, k.dlogits);
    if (!counts(k.t, r)) {
        if (lane == 0) {
            if (k.logp) k.logp[r] = 0.0;
            if (k.logp32) k.logp32[r] = 0.f;
            if (k.row_loss) k.row_loss[r] = 0.0;
            if (k.slope) k.slope[r] = 0.0;
            if (k.stats) k.stats[2 * r] = k.stats[2 * r + 1] = 0.f;
        }
        if (dx) write_zeros(dx, V, lane, 32, grads);
        return;
    }
    const Pieces<E> row(static_cast<const E*>(k.t.logits) + r * k.t.stride, V, logits_extent<E>(k.t));
    uint4 u[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) u[j] = row.load(j * 32 + lane);
    const int64_t said = k.t.ids[r];
    const int id = (uint64_t)said < (uint64_t)V ? (int)said : said < 0 ? 0 : V - 1;
    if (lane == 0 && id != said) atomicOr(&g_device_status, DEV_BAD_TOKEN);
    const float at = row.value(id);
    PolicyRow pr = {};
    if (k.policy) pr = policy_load(k.p, r);
    uint4 top4 = u[0];
#pragma unroll
    for (int j = 1; j < NV; ++j) top4 = piece_max<E>(top4, u[j]);
    const float M = warp_top(piece_top<E>(top4));
    const Ref ref(M);
    float e[SHORT_EPT], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) unpack<E>(u[j], e + j * N);
    exp_to_add<SHORT_EPT>(e, ref);
#pragma unroll
    for (int c = 0; c < SHORT_EPT; ++c) sum[c & 3] += e[c];
    float S = warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (M == -INFINITY) S = NAN;                   // no probabilities to speak of
    const double rel = relative(at, ref);
    PolicyTerms terms = {};
    float g = 0.f;
    if (k.policy) {
        terms = policy_terms(k.p, pr, rel, S);
        g = (float)(terms.slope * (inv_n * (double)k.scale));
    }
    if (lane == 0) {
        const double logp = rel - log((double)S);
        if (k.policy) k.row_loss[r] = terms.loss(k.p, pr, logp);
        if (k.slope) k.slope[r] = terms.slope;
        if (k.logp) k.logp[r] = logp;
        if (k.logp32) k.logp32[r] = (float)logp;
        if (k.stats) k.stats[2 * r] = M, k.stats[2 * r + 1] = 1.f / S;
    }
    if (!dx) return;
    __syncwarp();
    const float p = -g / S;
    const bool aligned = (reinterpret_cast<uintptr_t>(dx) & 15) == row.lead * sizeof(E);
#pragma unroll
    for (int j = 0; j < NV; ++j) write_piece<E, false>(row, e + j * N, j * 32 + lane, dx, aligned, p, grads);
    if (((id + row.lead) / N) % 32 == lane && grads.holds(dx + id)) dx[id] = from_f<E>(fmaf(p, exp_from(at, ref), g));   // (by the thread that wrote its piece)
}

struct DlogitsTask {
    ab_logit_rows t;
    const float *stats, *g, *scale;
    int64_t rows_per_g;
    void* dlogits;
    int blocks;      // per row
};
constexpr int DV = 4;   // pieces per thread of the gradient's kernel
template <class E>
__global__ void __launch_bounds__(LT, 6) dlogits_kernel(const __grid_constant__ DlogitsTask k) {
    constexpr int N = Pieces<E>::N;
    const int64_t r = blockIdx.x / k.blocks;
    const int V = k.t.vocab, blk = (int)(blockIdx.x - r * k.blocks), tid = threadIdx.x, at0 = blk * LT * DV;
    E* dx = static_cast<E*>(k.dlogits) + r * V;
    const Extent grads = grads_extent<E>(k.t, k.dlogits);
    if (!AB_BC(r < k.t.rows)) return;
    if (!counts(k.t, r)) {
        write_zeros(dx, V, blk * LT + tid, k.blocks * LT, grads);
        return;
    }
    const Pieces<E> row(static_cast<const E*>(k.t.logits) + r * k.t.stride, V, logits_extent<E>(k.t));
    const bool aligned = (reinterpret_cast<uintptr_t>(dx) & 15) == row.lead * sizeof(E);
    auto write = [&](auto whole) {
        constexpr bool FULL = decltype(whole)::value;
        uint4 u[DV];
#pragma unroll
        for (int j = 0; j < DV; ++j) u[j] = row.template get<FULL>(at0 + j * LT + tid);
        const int id = row_id(k.t, r);
        const float* gr = k.g + r / k.rows_per_g;
        const Extent all(k.g, (uint64_t)((k.t.rows + k.rows_per_g - 1) / k.rows_per_g) * sizeof(float));
        const float g = (all.holds(gr) ? *gr : 0.f) * (k.scale ? *k.scale : 1.f), p = -g * k.stats[2 * r + 1];
        const Ref ref(k.stats[2 * r]);
        const int own = (id + row.lead) / N - at0;
        const bool mine = own >= 0 && own < LT * DV && own % LT == tid;
        const float x_id = mine ? row.value(id) : 0.f;
#pragma unroll
        for (int j = 0; j < DV; ++j) {
            float e[N];
            unpack<E>(u[j], e);
            exp_from<N>(e, ref);
            write_piece<E, FULL>(row, e, at0 + j * LT + tid, dx, aligned, p, grads);
        }
        if (mine && grads.holds(dx + id)) dx[id] = from_f<E>(fmaf(p, exp_from(x_id, ref), g));
    };
    if (aligned && row.all_whole(at0, at0 + LT * DV)) write(std::true_type());
    else write(std::false_type());
}

constexpr int JT = 1024;

__device__ __forceinline__ double block_sum_jt(double v, double* red) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < JT / 32; ++i) t += red[i];
    return t;
}

// 1 / what the rows' losses are divided by
__device__ __forceinline__ double policy_inv_denom(const uint8_t* mask, int64_t rows, float denom, double* red) {
    if (denom != 0.f) return 1.0 / (double)denom;
    int n = 0;
    for (int64_t r = threadIdx.x; r < rows; r += JT) n += !mask || mask[r] ? 1 : 0;
    return 1.0 / fmax(block_sum_jt((double)n, red), 1.0);
}
__global__ void __launch_bounds__(JT) policy_denom_kernel(const uint8_t* mask, int64_t rows, float denom, double* inv) {
    __shared__ double red[JT / 32];
    const double d = policy_inv_denom(mask, rows, denom, red);
    if (threadIdx.x == 0) *inv = d;
}
// the loss, and the derivatives by the rows' log-probabilities divided as it is
__global__ void __launch_bounds__(JT) policy_join_kernel(const uint8_t* mask, float denom, const double* row_loss, const double* slope, int64_t rows, float* loss, float* g) {
    __shared__ double red[JT / 32];
    const double inv = policy_inv_denom(mask, rows, denom, red);
    pdl_wait();
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += JT) {
        s += row_loss[r];
        if (g) g[r] = (float)(slope[r] * inv);
    }
    s = block_sum_jt(s, red);
    if (threadIdx.x == 0) *loss = (float)(s * inv);
}

// sums of each answer's log-probabilities, the pairs' mean loss, its derivatives by the sums
__global__ void __launch_bounds__(JT) preference_join_kernel(const double* logp, int64_t pairs, int64_t steps, const float* ref, float beta,
                                                             float smoothing, float* loss, float* logp32, float* g) {
    __shared__ double red[JT / 32];
    double total = 0.0;
    pdl_wait();
    for (int64_t i = 0; i < pairs; ++i) {
        double side[2];
        for (int w = 0; w < 2; ++w) {
            double s = 0.0;
            for (int64_t t = threadIdx.x; t < steps; t += JT) {
                const double* p = logp + (i + w * pairs) * steps + t;
                s += Extent(logp, (uint64_t)(2 * pairs * steps) * sizeof(double)).holds(p) ? *p : 0.0;
            }
            side[w] = block_sum_jt(s, red);
        }
        const double m = (double)beta * ((side[0] - (double)ref[i]) - (side[1] - (double)ref[pairs + i]));
        // -log sigmoid(m) and -log sigmoid(-m) = that + m
        const double nls = log1p(exp(-fabs(m))) + fmax(-m, 0.0), sm = (double)smoothing;
        total += (1.0 - sm) * nls + sm * (nls + m);
        if (threadIdx.x == 0) {
            const double d = (double)beta * (sm - 1.0 / (1.0 + exp(m))) / (double)pairs;
            logp32[i] = (float)side[0];
            logp32[pairs + i] = (float)side[1];
            if (g) {
                g[i] = (float)d;
                g[pairs + i] = (float)-d;
            }
        }
    }
    if (threadIdx.x == 0) *loss = (float)(total / (double)pairs);
}

template <class F>
int with_type(int dtype, F f) {
    return dtype == AB_DT_F16 ? f(__half()) : dtype == AB_DT_BF16 ? f(__nv_bfloat16()) : f(0.f);
}

// pieces of the longest of the rows
template <class E>
int64_t row_pieces(const ab_logit_rows& t) {
    constexpr int N = 16 / sizeof(E);
    const bool on_boundaries = reinterpret_cast<uintptr_t>(t.logits) % 16 == 0 && (t.rows <= 1 || t.stride % N == 0);
    return (t.vocab + (on_boundaries ? 0 : N - 1) + N - 1) / N;
}

// Blocks per row, and values per thread. Long rows take as few blocks as hold them with 32 values a thread; few rows are spread over more blocks.
struct RowShape {
    int cluster, ept;
};
RowShape row_shape(int64_t rows, int64_t values, int n_sm) {
    RowShape s = {1, 8};
    while (s.cluster < MAX_CLUSTER && (values > (int64_t)s.cluster * LT * 32 || (rows * s.cluster < n_sm && values > (int64_t)s.cluster * LT * 8))) s.cluster *= 2;
    while (s.ept < 32 && values > (int64_t)s.cluster * LT * s.ept) s.ept *= 2;
    return s;
}

// what waits for its predecessor only where it reads its results
template <class... P, class... A>
int launch_behind(void (*kernel)(P...), int threads, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...), "join of a loss");
}

int logit_rows(const RowTask& k, cudaStream_t st) {
    if (!k.t.rows) return OK;
    return with_type(k.t.dtype, [&](auto e) -> int {
        using E = decltype(e);
        constexpr int N = Pieces<E>::N;
        const int n_sm = current_sm_count();
        const int64_t values = row_pieces<E>(k.t) * N;
        if (values <= 32 * SHORT_EPT) {
            logit_short_kernel<E><<<(unsigned)((k.t.rows + LW - 1) / LW), LT, 0, st>>>(k);
            return check_cuda(cudaGetLastError(), "rows of logits");
        }
        // The ring where a row would take more than two blocks of a cluster, and every SM has one. Ring and cluster, us, policy loss with gradient,
        // every row counting, fp16: 4096 x 65536 269 and 372, 1000 x 65536 76 and 100, 4096 x 32003 172 and 204, 4096 x 20011 166 and 189, 148 x
        // 65536 19 and 21; on the other side 4096 x 16384 109 and 95, 4096 x 9001 114 and 97, 100 x 65536 19 and 19. fp32: 4096 x 32003 206 and 241,
        // 1000 x 16384 39 and 35.
        if (values > 2 * LT * 32 && k.t.rows >= n_sm) {
            static PerDeviceOnce once;
            const int st_ = once.run(nullptr, [&](const DeviceProps&) -> int {
                AB_CUDA(cudaFuncSetAttribute(logit_ring_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_SLOTS * RING_CHUNK));
                return OK;
            });
            if (st_ != OK) return st_;
            logit_ring_kernel<E><<<(unsigned)k.t.rows, RING_THREADS, RING_SLOTS * RING_CHUNK, st>>>(k);
            return check_cuda(cudaGetLastError(), "rows of logits");
        }
        const RowShape s = row_shape(k.t.rows, values, n_sm);
        AB_CHECK_ARG(k.t.rows * s.cluster <= INT32_MAX, "too many rows of logits");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(k.t.rows * s.cluster));
        cfg.blockDim = dim3(LT);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = s.cluster;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        auto kernel = s.ept == 8 ? logit_rows_kernel<E, 8> : s.ept == 16 ? logit_rows_kernel<E, 16> : logit_rows_kernel<E, 32>;
        return check_cuda(cudaLaunchKernelEx(&cfg, kernel, k), "rows of logits");
    });
}

}  // namespace

int token_logp_fwd(const ab_logit_rows& t, double* logp, float* logp32, float* stats, cudaStream_t st) {
    RowTask k = {};
    k.t = t;
    k.logp = logp;
    k.logp32 = logp32;
    k.stats = stats;
    return logit_rows(k, st);
}

int token_logp_bwd(const ab_logit_rows& t, const float* stats, const float* g, int64_t rows_per_g, const float* scale, void* dlogits, cudaStream_t st) {
    if (!t.rows) return OK;
    return with_type(t.dtype, [&](auto e) -> int {
        const int64_t pieces = row_pieces<decltype(e)>(t);
        const int blocks = (int)((pieces + LT * DV - 1) / (LT * DV));
        AB_CHECK_ARG(t.rows * blocks <= INT32_MAX, "ab_token_logp_bwd: too many rows");
        const DlogitsTask k = {t, stats, g, scale, rows_per_g, dlogits, blocks};
        dlogits_kernel<decltype(e)><<<(unsigned)(t.rows * blocks), LT, 0, st>>>(k);
        return check_cuda(cudaGetLastError(), "ab_token_logp_bwd");
    });
}

int policy_loss(const ab_logit_rows& t, const ab_policy& p, float scale, float* loss, float* logp32, float* stats, float* g, void* dlogits,
                double* rows_scratch, cudaStream_t st) {
    // Where the gradient is made in this pass each block needs the denominator: it counts the rows itself up to 16384 of them (64 values a thread,
    // from L2, beside its row), a launch ahead of it does beyond that. rows_scratch: the rows' losses, that, and the rows' slopes.
    double* inv = nullptr;
    if (dlogits && (p.denom != 0.f || t.rows > 16384)) {
        inv = rows_scratch + t.rows;
        policy_denom_kernel<<<1, JT, 0, st>>>(t.mask, t.rows, p.denom, inv);
    }
    RowTask k = {};
    k.t = t;
    k.policy = 1;
    k.p = p;
    k.row_loss = rows_scratch;
    k.logp32 = logp32;
    k.stats = stats;
    k.slope = g ? rows_scratch + t.rows + 1 : nullptr;
    k.dlogits = dlogits;
    k.inv_denom = inv;
    k.scale = scale;
    const int s = logit_rows(k, st);
    if (s != OK) return s;
    return launch_behind(policy_join_kernel, JT, st, t.mask, p.denom, rows_scratch, k.slope, t.rows, loss, g);
}

int preference_loss(const ab_logit_rows& t, int64_t pairs, int64_t steps, const float* ref, float beta, float smoothing, float* loss, float* logp32,
                    float* stats, float* g, double* rows_scratch, cudaStream_t st) {
    const int s = token_logp_fwd(t, rows_scratch, nullptr, stats, st);
    if (s != OK) return s;
    return launch_behind(preference_join_kernel, JT, st, rows_scratch, pairs, steps, ref, beta, smoothing, loss, logp32, g);
}

}  // namespace ab
