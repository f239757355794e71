// C entries of the operators with gradients, of the gradient norm and of what serves a token: arguments checked, then the launchers of wkv_train.cu,
// norm.cu, loss.cu, clip.cu, sample.cu and int4.cu.
#include <algorithm>
#include <exception>
#include <vector>

#include "train.cuh"

namespace ab {
namespace {

bool is_16bit(int dtype) { return dtype == AB_DT_F16 || dtype == AB_DT_BF16; }
int elem_bytes(int dtype) { return dtype == AB_DT_F32 ? 4 : 2; }
bool on_boundary(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_seq(const ab_wkv7_seq* s, const char* who) {
    AB_CHECK_ARG(s, "%s: null pointer", who);
    AB_CHECK_ARG(is_16bit(s->dtype), "%s: dtype %d is neither fp16 nor bf16", who, s->dtype);
    AB_CHECK_ARG(s->B > 0 && s->T >= 0 && s->H > 0, "%s: bad shape (B=%d T=%d H=%d)", who, s->B, s->T, s->H);
    AB_CHECK_ARG((int64_t)s->B * s->H <= INT32_MAX && s->T <= INT32_MAX - 64, "%s: too many heads or steps", who);
    for (int i = 0; i < 6; ++i) {
        AB_CHECK_ARG(s->x[i] || s->T == 0, "%s: null pointer", who);
        AB_CHECK_ARG(on_boundary(s->x[i], 16) && s->batch_stride[i] % 8 == 0 && s->step_stride[i] % 8 == 0, "%s: inputs and their steps must start on 16-byte boundaries", who);
    }
    AB_CHECK_ARG(on_boundary(s->state, 16) && on_boundary(s->checkpoints, 16), "%s: states must start on a 16-byte boundary", who);
    AB_CHECK_ARG(on_boundary(s->lengths, 4), "%s: lengths must start on a 4-byte boundary", who);
    return OK;
}

int check_norm(int dtype, int wtype, int64_t rows, int C, int groups, int64_t x_stride, const char* who) {
    AB_CHECK_ARG(is_16bit(dtype) || dtype == AB_DT_F32, "%s: bad dtype %d", who, dtype);
    AB_CHECK_ARG(wtype == dtype || wtype == AB_DT_F32, "%s: weights of type %d beside rows of type %d", who, wtype, dtype);
    AB_CHECK_ARG(rows >= 0 && C > 0 && groups > 0 && C % groups == 0, "%s: bad shape (C=%d groups=%d)", who, C, groups);
    AB_CHECK_ARG(rows <= (int64_t)1 << 40 && x_stride >= 0, "%s: bad number of rows or stride", who);
    return OK;
}

int check_rows(const ab_logit_rows* t, const char* who) {
    AB_CHECK_ARG(t, "%s: null pointer", who);
    AB_CHECK_ARG(is_16bit(t->dtype) || t->dtype == AB_DT_F32, "%s: bad dtype %d", who, t->dtype);
    AB_CHECK_ARG(t->rows >= 0 && t->rows <= INT32_MAX && t->vocab > 0, "%s: bad shape", who);
    AB_CHECK_ARG(t->stride >= t->vocab || t->rows <= 1, "%s: rows of logits overlap", who);
    AB_CHECK_ARG(t->rows == 0 || (t->logits && t->ids), "%s: null pointer", who);
    AB_CHECK_ARG(on_boundary(t->logits, elem_bytes(t->dtype)) && on_boundary(t->ids, 8), "%s: misaligned pointer", who);
    return OK;
}

// the gradient may take the logits' own place, value for value; any other overlap overwrites what another row still reads
int check_in_place(const ab_logit_rows* t, const void* dlogits, const char* who) {
    if (t->rows == 0 || (dlogits == t->logits && (t->rows == 1 || t->stride == t->vocab))) return OK;
    const uintptr_t in = reinterpret_cast<uintptr_t>(t->logits), out = reinterpret_cast<uintptr_t>(dlogits);
    const uint64_t bytes = elem_bytes(t->dtype), in_bytes = ((uint64_t)(t->rows - 1) * t->stride + t->vocab) * bytes, out_bytes = (uint64_t)t->rows * t->vocab * bytes;
    AB_CHECK_ARG(out >= in + in_bytes || in >= out + out_bytes, "%s: the gradient overlaps the logits; in place only where the rows are dense", who);
    return OK;
}

int check_policy(const ab_policy* p, const ab_logit_rows& t, const void* scratch, const char* who) {
    AB_CHECK_ARG(p && scratch, "%s: null pointer", who);
    AB_CHECK_ARG(p->advantages || t.rows == 0, "%s: no advantages", who);
    AB_CHECK_ARG(p->clip_low >= 0.f && p->clip_low <= 1.f && p->clip_high >= 0.f, "%s: bad clip range", who);
    AB_CHECK_ARG(p->denom >= 0.f, "%s: the denominator is negative or not a number", who);
    return OK;
}

// Outputs that lie on one another, or on gradients other than their own, would be read and written in any order.
struct GradSpan {
    uintptr_t from, to;
    int64_t i;
    bool operator<(const GradSpan& o) const { return from < o.from; }
};
void in_order(std::vector<GradSpan>& v) {
    if (!std::is_sorted(v.begin(), v.end())) std::sort(v.begin(), v.end());
}
int check_apart(const ab_grad* t, int64_t n) {
    std::vector<GradSpan> out, in;
    out.reserve(n);
    for (int64_t i = 0; i < n; ++i) {
        if (t[i].n == 0) continue;
        const uintptr_t o = reinterpret_cast<uintptr_t>(t[i].out), g = reinterpret_cast<uintptr_t>(t[i].g);
        out.push_back({o, o + (uintptr_t)t[i].n * elem_bytes(t[i].out_dtype), i});
        if (o != g || elem_bytes(t[i].dtype) != elem_bytes(t[i].out_dtype)) in.push_back({g, g + (uintptr_t)t[i].n * elem_bytes(t[i].dtype), i});
    }
    in_order(out);
    for (size_t i = 1; i < out.size(); ++i)
        AB_CHECK_ARG(out[i].from >= out[i - 1].to, "ab_clip_grad_norm: outputs %lld and %lld overlap", (long long)out[i - 1].i, (long long)out[i].i);
    in_order(in);
    size_t at = 0;
    for (const GradSpan& s : in) {   // (outputs do not overlap: their ends are in order too. A later s begins no earlier, so what ends before this one is done with)
        while (at < out.size() && out[at].to <= s.from) ++at;
        AB_CHECK_ARG(at == out.size() || out[at].from >= s.to, "ab_clip_grad_norm: output %lld overlaps gradient %lld", (long long)out[at].i, (long long)s.i);
    }
    return OK;
}

}  // namespace
}  // namespace ab

using namespace ab;

#define AB_CHECK(call)             \
    do {                           \
        const int _c = (call);     \
        if (_c != OK) return _c;   \
    } while (0)

extern "C" {

size_t ab_wkv7_checkpoint_bytes(const ab_wkv7_seq* s) {
    if (!s || s->B <= 0 || s->T < 0 || s->H <= 0) return 0;
    return (size_t)s->B * s->H * (size_t)((s->T + WKV_CHUNK - 1) / WKV_CHUNK) * 4096 * sizeof(float);
}

int ab_wkv7_seq_fwd(const ab_wkv7_seq* s, void* y, float* state_out, void* stream) {
    AB_CHECK(check_seq(s, "ab_wkv7_seq_fwd"));
    AB_CHECK_ARG((y || s->T == 0) && state_out, "ab_wkv7_seq_fwd: null pointer");
    AB_CHECK_ARG(on_boundary(y, 16) && on_boundary(state_out, 16), "ab_wkv7_seq_fwd: outputs must start on a 16-byte boundary");
    return wkv_train_fwd(*s, y, state_out, (cudaStream_t)stream);
}

int ab_wkv7_seq_bwd(const ab_wkv7_seq* s, const void* dy, int64_t dy_batch_stride, int64_t dy_step_stride, const float* dstate_out,
                    void* const* dx, float* dstate, void* stream) {
    AB_CHECK(check_seq(s, "ab_wkv7_seq_bwd"));
    AB_CHECK_ARG(dx, "ab_wkv7_seq_bwd: null pointer");
    AB_CHECK_ARG(s->checkpoints || s->T == 0, "ab_wkv7_seq_bwd: needs the checkpoints of the forward pass");
    AB_CHECK_ARG(!dy || (on_boundary(dy, 16) && dy_batch_stride % 8 == 0 && dy_step_stride % 8 == 0), "ab_wkv7_seq_bwd: dy and its steps must start on 16-byte boundaries");
    AB_CHECK_ARG(on_boundary(dstate_out, 16) && on_boundary(dstate, 16), "ab_wkv7_seq_bwd: misaligned pointer");
    WkvBackward g = {dy, dy_batch_stride, dy_step_stride, dstate_out, {}, dstate};
    for (int i = 0; i < 6; ++i) {
        AB_CHECK_ARG(on_boundary(dx[i], 16), "ab_wkv7_seq_bwd: gradients must start on a 16-byte boundary");
        g.dx[i] = dx[i];
    }
    return wkv_train_bwd(*s, g, (cudaStream_t)stream);
}

int ab_layer_norm_fwd(int dtype, int wtype, int64_t rows, int C, int groups, const void* x, int64_t x_stride, const void* w, const void* b,
                      float eps, void* y, float* mean, float* rstd, void* stream) {
    AB_CHECK(check_norm(dtype, wtype, rows, C, groups, x_stride, "ab_layer_norm_fwd"));
    if (rows == 0) return OK;
    AB_CHECK_ARG(x && y && (mean != nullptr) == (rstd != nullptr), "ab_layer_norm_fwd: null pointer");
    AB_CHECK_ARG(on_boundary(x, elem_bytes(dtype)) && on_boundary(y, elem_bytes(dtype)) && on_boundary(w, elem_bytes(wtype)) &&
                 on_boundary(b, elem_bytes(wtype)), "ab_layer_norm_fwd: misaligned pointer");
    NormArgs a = {};
    a.dtype = dtype; a.wtype = wtype; a.C = C; a.groups = groups; a.rows = rows; a.x_stride = x_stride; a.eps = eps;
    a.x = x; a.w = w; a.b = b; a.y = y; a.mean = mean; a.rstd = rstd;
    return layer_norm_fwd(a, (cudaStream_t)stream);
}

size_t ab_layer_norm_scratch_bytes(int64_t rows, int C) { return rows < 0 || C <= 0 ? 0 : layer_norm_scratch_bytes(rows, C); }

int ab_layer_norm_bwd(int dtype, int wtype, int64_t rows, int C, int groups, const void* x, int64_t x_stride, const void* w, const float* mean,
                      const float* rstd, const void* dy, int64_t dy_stride, void* dx, void* dw, void* db, void* scratch, void* stream) {
    AB_CHECK(check_norm(dtype, wtype, rows, C, groups, x_stride, "ab_layer_norm_bwd"));
    AB_CHECK_ARG(rows == 0 || (x && dy && mean && rstd), "ab_layer_norm_bwd: null pointer");
    AB_CHECK_ARG(scratch || rows == 0 || !(dw || db), "ab_layer_norm_bwd: the weights' gradients need scratch");
    AB_CHECK_ARG(dy_stride >= 0, "ab_layer_norm_bwd: bad stride");
    AB_CHECK_ARG(on_boundary(x, elem_bytes(dtype)) && on_boundary(dy, elem_bytes(dtype)) && on_boundary(dx, elem_bytes(dtype)) &&
                 on_boundary(w, elem_bytes(wtype)) && on_boundary(dw, elem_bytes(wtype)) && on_boundary(db, elem_bytes(wtype)) &&
                 on_boundary(scratch, 16), "ab_layer_norm_bwd: misaligned pointer");
    NormArgs a = {};
    a.dtype = dtype; a.wtype = wtype; a.C = C; a.groups = groups; a.rows = rows; a.x_stride = x_stride; a.dy_stride = dy_stride;
    a.x = x; a.w = w; a.dy = dy; a.dx = dx; a.dw = dw; a.db = db;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.scratch = static_cast<float*>(scratch);
    a.scratch_bytes = (int64_t)layer_norm_scratch_bytes(rows, C);
    return layer_norm_bwd(a, (cudaStream_t)stream);
}

int ab_token_logp_fwd(const ab_logit_rows* t, double* logp, float* logp32, float* stats, void* stream) {
    AB_CHECK(check_rows(t, "ab_token_logp_fwd"));
    AB_CHECK_ARG(logp || logp32 || t->rows == 0, "ab_token_logp_fwd: null pointer");
    return token_logp_fwd(*t, logp, logp32, stats, (cudaStream_t)stream);
}

int ab_token_logp_bwd(const ab_logit_rows* t, const float* stats, const float* g, int64_t rows_per_g, const float* scale, void* dlogits,
                      void* stream) {
    AB_CHECK(check_rows(t, "ab_token_logp_bwd"));
    AB_CHECK_ARG(t->rows == 0 || (stats && g && dlogits), "ab_token_logp_bwd: null pointer");
    AB_CHECK_ARG(rows_per_g > 0, "ab_token_logp_bwd: bad number of rows per gradient");
    AB_CHECK(check_in_place(t, dlogits, "ab_token_logp_bwd"));
    return token_logp_bwd(*t, stats, g, rows_per_g, scale, dlogits, (cudaStream_t)stream);
}

int ab_policy_loss_fwd(const ab_logit_rows* t, const ab_policy* p, float* loss, float* logp32, float* stats, float* g, double* rows_scratch,
                       void* stream) {
    AB_CHECK(check_rows(t, "ab_policy_loss_fwd"));
    AB_CHECK(check_policy(p, *t, rows_scratch, "ab_policy_loss_fwd"));
    AB_CHECK_ARG(loss && (logp32 || t->rows == 0), "ab_policy_loss_fwd: null pointer");
    return policy_loss(*t, *p, 1.f, loss, logp32, stats, g, nullptr, rows_scratch, (cudaStream_t)stream);
}

int ab_policy_loss_grad(const ab_logit_rows* t, const ab_policy* p, float scale, float* loss, float* logp32, void* dlogits,
                        double* rows_scratch, void* stream) {
    AB_CHECK(check_rows(t, "ab_policy_loss_grad"));
    AB_CHECK(check_policy(p, *t, rows_scratch, "ab_policy_loss_grad"));
    AB_CHECK_ARG(loss && ((logp32 && dlogits) || t->rows == 0), "ab_policy_loss_grad: null pointer");
    AB_CHECK(check_in_place(t, dlogits, "ab_policy_loss_grad"));
    return policy_loss(*t, *p, scale, loss, logp32, nullptr, nullptr, dlogits, rows_scratch, (cudaStream_t)stream);
}

int ab_preference_loss_fwd(const ab_logit_rows* t, int64_t pairs, int64_t steps, const float* ref_logp, float beta, float smoothing, float* loss,
                           float* logp32, float* stats, float* g, double* rows_scratch, void* stream) {
    AB_CHECK(check_rows(t, "ab_preference_loss_fwd"));
    AB_CHECK_ARG(pairs > 0 && steps >= 0 && pairs <= INT32_MAX && steps <= INT32_MAX && 2 * pairs * steps == t->rows, "ab_preference_loss_fwd: bad shape");
    AB_CHECK_ARG(ref_logp && loss && logp32 && (rows_scratch || t->rows == 0), "ab_preference_loss_fwd: null pointer");
    AB_CHECK_ARG(smoothing >= 0.f && smoothing <= 1.f, "ab_preference_loss_fwd: smoothing outside 0 .. 1");
    return preference_loss(*t, pairs, steps, ref_logp, beta, smoothing, loss, logp32, stats, g, rows_scratch, (cudaStream_t)stream);
}

size_t ab_clip_grad_norm_scratch_bytes(int64_t tensors) { return tensors < 0 ? 0 : clip_scratch_bytes(tensors); }

int ab_clip_grad_norm(const ab_grad* t, int64_t tensors, double scale, double max_norm, float* norm, void* scratch, void* stream) {
    AB_CHECK_ARG(tensors >= 0 && (t || tensors == 0) && norm && scratch, "ab_clip_grad_norm: null pointer, or a negative number of tensors");
    AB_CHECK_ARG(on_boundary(scratch, 8) && on_boundary(norm, 4), "ab_clip_grad_norm: misaligned pointer");
    AB_CHECK_ARG(scale > 0 && (float)scale < INFINITY, "ab_clip_grad_norm: the scale must be positive and finite, in 32 bits");
    AB_CHECK_ARG(max_norm >= 0, "ab_clip_grad_norm: the largest norm is negative or not a number");
    bool with = false, without = false;
    for (int64_t i = 0; i < tensors; ++i) {
        const ab_grad& e = t[i];
        AB_CHECK_ARG((is_16bit(e.dtype) || e.dtype == AB_DT_F32) && (is_16bit(e.out_dtype) || e.out_dtype == AB_DT_F32), "ab_clip_grad_norm: tensor %lld has a bad dtype", (long long)i);
        AB_CHECK_ARG(e.n >= 0 && e.n <= (int64_t)1 << 40 && (e.g || e.n == 0), "ab_clip_grad_norm: tensor %lld has a bad size or no values", (long long)i);
        AB_CHECK_ARG(on_boundary(e.g, elem_bytes(e.dtype)) && on_boundary(e.out, elem_bytes(e.out_dtype)), "ab_clip_grad_norm: tensor %lld is misaligned", (long long)i);
        if (e.n > 0) (e.out ? with : without) = true;
    }
    AB_CHECK_ARG(!(with && without), "ab_clip_grad_norm: outputs for some tensors only");
    if (with) {
        try {
            AB_CHECK(check_apart(t, tensors));
        } catch (const std::exception&) {
            set_error("ab_clip_grad_norm: out of host memory");
            return ERR_TOO_LARGE;
        }
    }
    return clip_grad_norm(t, tensors, with, scale, max_norm, norm, static_cast<double*>(scratch), (cudaStream_t)stream);
}

int ab_linear_int4(const ab_int4* m, int rows, const void* x, int64_t x_stride, void* y, void* stream) {
    AB_CHECK_ARG(m, "ab_linear_int4: null pointer");
    AB_CHECK_ARG(is_16bit(m->dtype), "ab_linear_int4: dtype %d is neither fp16 nor bf16", m->dtype);
    AB_CHECK_ARG(rows >= 0 && m->n_out > 0 && m->k > 0 && x_stride >= 0, "ab_linear_int4: bad shape (rows=%d n_out=%d k=%d)", rows, m->n_out, m->k);
    AB_CHECK_ARG((m->group == 32 || m->group == 64 || (m->group > 0 && m->group % 128 == 0)) && m->k % m->group == 0,
                 "ab_linear_int4: groups of %d inputs (32, 64 or a multiple of 128, which divides %d)", m->group, m->k);
    AB_CHECK_ARG(rows <= 65535, "ab_linear_int4: %d rows are too many (65535 at most: each 16 of them read the matrix once more)", rows);
    if (rows == 0) return OK;
    AB_CHECK_ARG(m->w && m->scale && x && y, "ab_linear_int4: null pointer");
    AB_CHECK_ARG(on_boundary(m->w, 16), "ab_linear_int4: the codes must start on a 16-byte boundary");
    AB_CHECK_ARG(on_boundary(m->scale, 2) && on_boundary(x, 2) && on_boundary(y, 2), "ab_linear_int4: misaligned pointer");
    return linear_int4(*m, rows, x, x_stride, y, (cudaStream_t)stream);
}

int ab_sample_filtered(int dtype, int64_t rows, int vocab, const void* logits, int64_t stride, const float* uniform, const ab_sampling* p,
                       int64_t* ids, float* logp, void* stream) {
    AB_CHECK_ARG(p, "ab_sample_filtered: null pointer");
    AB_CHECK_ARG(is_16bit(dtype) || dtype == AB_DT_F32, "ab_sample_filtered: bad dtype %d", dtype);
    AB_CHECK_ARG(rows >= 0 && vocab > 0 && vocab <= 1 << 18 && stride >= 0, "ab_sample_filtered: bad shape (a vocabulary of up to 2^18)");
    AB_CHECK_ARG(p->temperature || p->temperature_all >= 0, "ab_sample_filtered: the temperature is negative or not a number");
    AB_CHECK_ARG((p->top_p || p->top_p_all >= 0) && (p->min_p || p->min_p_all >= 0), "ab_sample_filtered: top_p or min_p is negative or not a number");
    if (rows == 0) return OK;
    AB_CHECK_ARG(logits && uniform && ids && logp, "ab_sample_filtered: null pointer");
    AB_CHECK_ARG(on_boundary(logits, elem_bytes(dtype)) && on_boundary(uniform, 4) && on_boundary(ids, 8) && on_boundary(logp, 4) && on_boundary(p->temperature, 4) &&
                 on_boundary(p->top_p, 4) && on_boundary(p->min_p, 4) && on_boundary(p->top_k, 4), "ab_sample_filtered: misaligned pointer");
    return sample_filtered(dtype, rows, vocab, logits, stride, uniform, *p, ids, logp, (cudaStream_t)stream);
}

}  // extern "C"
