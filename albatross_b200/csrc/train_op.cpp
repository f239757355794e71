// The operators with gradients as torch operators (torch.ops.albatross_b200.*): arguments checked, memory from torch's allocator, the C entries of
// the kernel library called on torch's current stream of the tensors' device, gradients through torch's C++ autograd. In Python the same costs 100 us
// a training pass more than the engine's own 50, which is what small calls take.
//
// The kernel library is not linked: albatross_b200_train_bind() is given the path of the one that the package has loaded (the normal or the
// range-checking build).
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>

#include "op.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
#define AB_ENTRY(name) decltype(&::name) name = nullptr
    AB_ENTRY(ab_last_error);
    AB_ENTRY(ab_wkv7_checkpoint_bytes);
    AB_ENTRY(ab_wkv7_seq_fwd);
    AB_ENTRY(ab_wkv7_seq_bwd);
    AB_ENTRY(ab_layer_norm_fwd);
    AB_ENTRY(ab_layer_norm_scratch_bytes);
    AB_ENTRY(ab_layer_norm_bwd);
    AB_ENTRY(ab_token_logp_fwd);
    AB_ENTRY(ab_token_logp_bwd);
    AB_ENTRY(ab_policy_loss_fwd);
    AB_ENTRY(ab_policy_loss_grad);
    AB_ENTRY(ab_preference_loss_fwd);
    AB_ENTRY(ab_clip_grad_norm_scratch_bytes);
    AB_ENTRY(ab_clip_grad_norm);
#undef AB_ENTRY
} lib;

// (Backward passes take their saved tensors before they go below autograd: unpacking one may recompute the forward pass, which has to be recorded.)
// What a backward pass refuses. Gradients are not differentiable: asking for a graph of them is an error, not a silent zero. And in a stream capture
// a leaf that an earlier graph still ties to the default stream: adding its gradient would make that stream wait for the capturing one, which the
// default stream cannot, and the capture would be lost with a less telling error.
void check_backward(const variable_list& grads) {
    for (const Tensor& g : grads) check_plain("albatross_b200: gradients", g);
    TORCH_CHECK(!at::GradMode::is_enabled(), "albatross_b200: the gradients of these operators cannot be differentiated again (create_graph)");
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const torch::autograd::Edge& e = node->next_edge(i);
        if (!node->task_should_compute_output(i)) continue;   // its gradient is not asked for: nothing waits
        if (!e.function || !dynamic_cast<torch::autograd::AccumulateGrad*>(e.function.get())) continue;
        const auto s = e.function->stream();
        TORCH_CHECK(!s || at::cuda::CUDAStream(*s).stream() != nullptr,
                    "albatross_b200: a gradient is captured into a CUDA graph while an earlier autograd graph of the same leaf, made on the default stream, still lives; release that one first");
    }
}

// ---- the recurrence ----------------------------------------------------------------------------------------------------------------
// [B, T, C] with a dense last dimension and every step on a 16-byte boundary; others are copied
Tensor steps(const Tensor& t) {
    if (t.stride(2) == 1 && ((t.stride(0) | t.stride(1)) & 7) == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}
// a state, dense and on a 16-byte boundary (a view into a larger tensor need not be)
Tensor dense_state(const Tensor& t) {
    const Tensor d = t.contiguous();
    return (reinterpret_cast<uintptr_t>(d.data_ptr()) & 15) == 0 ? d : d.clone();
}
ab_wkv7_seq seq_of(const Tensor* x, const Tensor& state, const Tensor& lengths, const Tensor& checkpoints) {
    ab_wkv7_seq s = {};
    s.dtype = type_of(x[0]);
    s.B = (int32_t)x[0].size(0), s.T = (int32_t)x[0].size(1), s.H = (int32_t)(x[0].size(2) / 64);
    for (int i = 0; i < 6; ++i) {
        s.x[i] = x[i].data_ptr();
        s.batch_stride[i] = x[i].stride(0), s.step_stride[i] = x[i].stride(1);
    }
    s.state = f32(state);
    s.lengths = lengths.defined() ? lengths.data_ptr<int32_t>() : nullptr;
    s.checkpoints = f32(checkpoints);
    return s;
}
std::pair<Tensor, Tensor> wkv_forward(const Tensor* x, const Tensor& state, const Tensor& lengths, Tensor* checkpoints) {
    const c10::cuda::CUDAGuard guard(x[0].device());
    const int64_t B = x[0].size(0), T = x[0].size(1), C = x[0].size(2);
    Tensor y = like({B, T, C}, x[0], x[0].scalar_type()), out = like({B, C / 64, 64, 64}, x[0], at::kFloat);
    if (checkpoints) {
        const ab_wkv7_seq s = seq_of(x, state, lengths, Tensor());
        *checkpoints = like({(int64_t)(lib.ab_wkv7_checkpoint_bytes(&s) / sizeof(float))}, x[0], at::kFloat);
    }
    const ab_wkv7_seq s = seq_of(x, state, lengths, checkpoints ? *checkpoints : Tensor());
    check(lib.ab_wkv7_seq_fwd(&s, y.data_ptr(), f32(out), stream()), "ab_wkv7_seq_fwd");
    return {y, out};
}
struct Wkv7 : torch::autograd::Function<Wkv7> {
    static variable_list forward(AutogradContext* ctx, Tensor r, Tensor w, Tensor k, Tensor v, Tensor a, Tensor b, OptTensor state_, Plain lengths_) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor state = given(state_), lengths = lengths_.t;
        const Tensor x[6] = {r, w, k, v, a, b};
        Tensor checkpoints;
        auto [y, out] = wkv_forward(x, state, lengths, &checkpoints);
        ctx->save_for_backward({state, r, w, k, v, a, b, lengths, checkpoints});
        ctx->set_materialize_grads(false);
        return {y, out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward(grads);
        const variable_list saved = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor* x = saved.data() + 1;
        const c10::cuda::CUDAGuard guard(x[0].device());
        const int64_t B = x[0].size(0), T = x[0].size(1), C = x[0].size(2);
        variable_list out(8);
        if (saved[0].defined() && ctx->needs_input_grad(6)) out[6] = like({B, C / 64, 64, 64}, x[0], at::kFloat);
        void* dx[6];
        for (int i = 0; i < 6; ++i) {
            if (ctx->needs_input_grad(i)) out[i] = like({B, T, C}, x[0], x[0].scalar_type());
            dx[i] = ptr(out[i]);
        }
        const Tensor dy = grads[0].defined() ? steps(grads[0]) : Tensor(), dout = grads[1].defined() ? dense_state(grads[1]) : Tensor();
        const ab_wkv7_seq s = seq_of(x, saved[0], saved[7], saved[8]);
        check(lib.ab_wkv7_seq_bwd(&s, ptr(dy), dy.defined() ? dy.stride(0) : 0, dy.defined() ? dy.stride(1) : 0, f32(dout), dx, f32(out[6]), stream()), "ab_wkv7_seq_bwd");
        return out;
    }
};
std::tuple<Tensor, Tensor> wkv7(const OptTensor& state_, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a, const Tensor& b, const OptTensor& lengths_) {
    check_plain("RWKV7_TRAIN_OP", given(state_), r, w, k, v, a, b, given(lengths_));
    TORCH_CHECK(r.dim() == 3 && r.is_cuda() && is_16bit(r), "RWKV7_TRAIN_OP: r must be [B, T, C], fp16 or bf16, on a CUDA device");
    const int64_t B = r.size(0), T = r.size(1), C = r.size(2);
    TORCH_CHECK(B > 0 && C > 0 && C % 64 == 0, "RWKV7_TRAIN_OP: heads are of 64 channels, got C = ", std::to_string(C));
    TORCH_CHECK(B * (C / 64) <= INT32_MAX && T <= INT32_MAX - 64, "RWKV7_TRAIN_OP: too many heads or steps");
    for (const Tensor* t : {&w, &k, &v, &a, &b})
        TORCH_CHECK(t->sizes() == r.sizes() && t->scalar_type() == r.scalar_type() && t->device() == r.device(), "RWKV7_TRAIN_OP: r, w, k, v, a, b differ in shape, type or device");
    Tensor state = given(state_), lengths = given(lengths_);
    if (state.defined()) {
        TORCH_CHECK(state.sizes() == at::IntArrayRef({B, C / 64, 64, 64}) && state.scalar_type() == at::kFloat && state.device() == r.device(),
                    "RWKV7_TRAIN_OP: the state must be fp32 [B, H, 64, 64] on the device of r");
        state = dense_state(state);
    }
    if (lengths.defined()) {
        TORCH_CHECK(lengths.sizes() == at::IntArrayRef({B}) && lengths.scalar_type() == at::kInt && lengths.device() == r.device(),
                    "RWKV7_TRAIN_OP: lengths must be int32 [B] on the device of r");
        lengths = lengths.contiguous();
    }
    const Tensor x[6] = {steps(r), steps(w), steps(k), steps(v), steps(a), steps(b)};
    if (needs_grad(state, x[0], x[1], x[2], x[3], x[4], x[5])) {
        const variable_list y = Wkv7::apply(x[0], x[1], x[2], x[3], x[4], x[5], or_none(state), Plain{lengths});
        return {y[0], y[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, out] = wkv_forward(x, state, lengths, nullptr);
    return {y, out};
}

// ---- the norms ---------------------------------------------------------------------------------------------------------------------
int weight_type(const Tensor& x, const Tensor& w, const Tensor& b) { return type_of(w.defined() ? w : b.defined() ? b : x); }
Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t groups, Tensor* stats) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor rows = as_rows(x);
    const int64_t n = rows.size(0), C = rows.size(1);
    Tensor y = like(x.sizes(), x, x.scalar_type());
    if (stats) *stats = like({2, n, groups}, x, at::kFloat);
    float* at_ = stats ? stats->data_ptr<float>() : nullptr;
    check(lib.ab_layer_norm_fwd(type_of(x), weight_type(x, w, b), n, (int)C, (int)groups, rows.data_ptr(), rows.stride(0), ptr(w), ptr(b), (float)eps, y.data_ptr(), at_,
                                at_ ? at_ + n * groups : nullptr, stream()), "ab_layer_norm_fwd");
    return y;
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, Tensor x, OptTensor w_, OptTensor b_, double eps, int64_t groups) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor w = given(w_), b = given(b_);
        Tensor stats;
        Tensor y = norm_forward(x, w, b, eps, groups, &stats);
        ctx->save_for_backward({x, w, b, stats});
        ctx->saved_data["groups"] = groups;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward(grads);
        const variable_list saved = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        const c10::cuda::CUDAGuard guard(x.device());
        const Tensor rows = as_rows(x), dy = as_rows(grads[0]);
        const int64_t n = rows.size(0), C = rows.size(1);
        variable_list out(5);
        if (ctx->needs_input_grad(0)) out[0] = like(x.sizes(), x, x.scalar_type());
        if (w.defined() && ctx->needs_input_grad(1)) out[1] = like({C}, w, w.scalar_type());
        if (b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1)) out[2] = like({C}, b, b.scalar_type());
        Tensor scratch;
        if (out[1].defined() || out[2].defined()) scratch = like({(int64_t)lib.ab_layer_norm_scratch_bytes(n, (int)C)}, x, at::kByte);
        const float* at_ = stats.data_ptr<float>();
        check(lib.ab_layer_norm_bwd(type_of(x), weight_type(x, w, b), n, (int)C, (int)groups, rows.data_ptr(), rows.stride(0), ptr(w), at_, at_ + n * groups, dy.data_ptr(), dy.stride(0),
                                    ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(scratch), stream()), "ab_layer_norm_bwd");
        return out;
    }
};
Tensor layer_norm(const Tensor& x_, const OptTensor& weight, const OptTensor& bias, double eps, int64_t groups) {
    check_plain("layer_norm", x_, given(weight), given(bias));
    TORCH_CHECK(x_.is_cuda() && is_known(x_) && x_.dim() >= 1, "layer_norm: x must be fp16, bf16 or fp32 on a CUDA device");
    const Tensor x = one_stride(x_, 0);
    const int64_t C = x.size(-1);
    TORCH_CHECK(C > 0 && C <= INT32_MAX && groups > 0 && C % groups == 0, "layer_norm: ", std::to_string(C), " values do not make ", std::to_string(groups), " groups");
    Tensor w = given(weight), b = given(bias);
    for (Tensor* t : {&w, &b})
        if (t->defined()) {
            TORCH_CHECK(t->sizes() == at::IntArrayRef({C}) && (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat) && t->device() == x.device(),
                        "layer_norm: weight and bias must be [C] of the type of x or fp32, on its device");
            *t = t->contiguous();
        }
    TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "layer_norm: weight and bias differ in type");
    if (needs_grad(x, w, b)) return LayerNorm::apply(x, or_none(w), or_none(b), eps, groups);
    at::AutoDispatchBelowADInplaceOrView below;
    return norm_forward(x, w, b, eps, groups, nullptr);
}

// ---- losses on logits ----------------------------------------------------------------------------------------------------------------
struct Rows {   // what a loss works on; the tensors that are kept for its gradient
    Tensor logits, ids, mask, rows;
    ab_logit_rows t = {};
    Rows(const Tensor& logits_, const Tensor& ids_, const Tensor& mask_) : logits(logits_), ids(ids_), mask(mask_), rows(as_rows(logits_)) {
        t.dtype = type_of(rows);
        t.vocab = (int32_t)rows.size(1);
        t.rows = rows.size(0), t.stride = rows.stride(0);
        t.logits = rows.data_ptr();
        t.ids = ids.data_ptr<int64_t>();
        t.mask = static_cast<const uint8_t*>(ptr(mask));
    }
};
void check_rows(const char* who, Tensor& logits, Tensor& ids, Tensor& mask) {
    TORCH_CHECK(logits.is_cuda() && is_known(logits) && logits.dim() >= 1 && logits.size(-1) > 0 && logits.size(-1) <= INT32_MAX, who,
                ": logits must be [..., V], fp16, bf16 or fp32, on a CUDA device");
    TORCH_CHECK(ids.sizes() == logits.sizes().slice(0, logits.dim() - 1) && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt) && ids.device() == logits.device(), who,
                ": ids must be int64 or int32 of the shape of logits without its last dimension, on its device");
    TORCH_CHECK(!mask.defined() || (mask.sizes() == ids.sizes() && mask.scalar_type() == at::kBool && mask.device() == logits.device()), who, ": mask must be bool of the ids' shape");
    logits = one_stride(logits, logits.size(-1));   // (rows that share their values, as expand() makes them, are copied too)
    ids = ids.to(at::kLong).contiguous();
    if (mask.defined()) mask = mask.contiguous();
}
Tensor dlogits_of(const Tensor& logits, const Tensor& ids, const Tensor& mask, const Tensor& stats, const Tensor& g, int64_t rows_per_g, const Tensor& scale) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const Rows r(logits, ids, mask);
    Tensor out = like(logits.sizes(), logits, logits.scalar_type());
    check(lib.ab_token_logp_bwd(&r.t, f32(stats), f32(g), rows_per_g, f32(scale), out.data_ptr(), stream()), "ab_token_logp_bwd");
    return out;
}
Tensor logp_forward(const Tensor& logits, const Tensor& ids, const Tensor& mask, Tensor* stats) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const Rows r(logits, ids, mask);
    Tensor logp = like(ids.sizes(), logits, at::kFloat);
    if (stats) *stats = like({r.t.rows, 2}, logits, at::kFloat);
    check(lib.ab_token_logp_fwd(&r.t, nullptr, f32(logp), stats ? f32(*stats) : nullptr, stream()), "ab_token_logp_fwd");
    return logp;
}
struct TokenLogp : torch::autograd::Function<TokenLogp> {
    static Tensor forward(AutogradContext* ctx, Tensor logits, Plain ids_, Plain mask_) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &ids = ids_.t, &mask = mask_.t;
        Tensor stats;
        Tensor logp = logp_forward(logits, ids, mask, &stats);
        ctx->save_for_backward({logits, ids, mask, stats});
        return logp;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward(grads);
        const variable_list s = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        return {dlogits_of(s[0], s[1], s[2], s[3], grads[0].contiguous(), 1, Tensor()), Tensor(), Tensor()};
    }
};
Tensor token_logp(const Tensor& logits_, const Tensor& ids_, const OptTensor& mask_) {
    Tensor logits = logits_, ids = ids_, mask = given(mask_);
    check_plain("token_logp", logits_, ids_, given(mask_));
    check_rows("token_logp", logits, ids, mask);
    if (needs_grad(logits)) return TokenLogp::apply(logits, Plain{ids}, Plain{mask});
    at::AutoDispatchBelowADInplaceOrView below;
    return logp_forward(logits, ids, mask, nullptr);
}

struct PolicyArgs {
    Tensor old_logp, advantages, ref_logp;
    ab_policy p = {};
};
PolicyArgs policy_args(const Tensor& logits, const Tensor& ids, const OptTensor& old_logp, const Tensor& advantages, const OptTensor& ref_logp, double low, double high, double kl,
                       double denom) {
    at::NoGradGuard no_grad;
    auto rows = [&](const Tensor& t) {
        if (!t.defined()) return t;
        TORCH_CHECK(t.device() == logits.device(), "policy_loss: old_logp, advantages and ref_logp must be on the device of logits");
        const Tensor f = t.scalar_type() == at::kFloat ? t : t.to(at::kFloat);
        return (f.sizes() == ids.sizes() ? f : f.broadcast_to(ids.sizes())).contiguous();
    };
    PolicyArgs a = {rows(given(old_logp)), rows(advantages), rows(given(ref_logp))};
    TORCH_CHECK(low >= 0 && low <= 1 && high >= 0, "policy_loss: bad clip range");
    TORCH_CHECK(denom == 0 || (float)denom > 0, "policy_loss: the denominator must be positive, in 32 bits too");   // 0 stands for the number of tokens
    a.p = {f32(a.old_logp), f32(a.advantages), f32(a.ref_logp), (float)low, (float)high, (float)kl, (float)denom};
    return a;
}
std::pair<Tensor, Tensor> policy_forward(const Tensor& logits, const Tensor& ids, const Tensor& mask, const PolicyArgs& a, Tensor* stats, Tensor* g) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const Rows r(logits, ids, mask);
    Tensor loss = like({}, logits, at::kFloat), logp = like(ids.sizes(), logits, at::kFloat), scratch = like({2 * r.t.rows + 1}, logits, at::kDouble);
    if (stats) *stats = like({r.t.rows, 2}, logits, at::kFloat), *g = like({r.t.rows}, logits, at::kFloat);
    check(lib.ab_policy_loss_fwd(&r.t, &a.p, f32(loss), f32(logp), stats ? f32(*stats) : nullptr, stats ? f32(*g) : nullptr, scratch.data_ptr<double>(), stream()), "ab_policy_loss_fwd");
    return {loss, logp};
}
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, Tensor logits, Plain ids_, Plain mask_, const PolicyArgs& a) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &ids = ids_.t, &mask = mask_.t;
        Tensor stats, g;
        auto [loss, logp] = policy_forward(logits, ids, mask, a, &stats, &g);
        ctx->save_for_backward({logits, ids, mask, stats, g});
        ctx->mark_non_differentiable({logp});
        return {loss, logp};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward(grads);
        const variable_list s = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        return {dlogits_of(s[0], s[1], s[2], s[3], s[4], 1, grads[0].contiguous()), Tensor(), Tensor(), Tensor()};
    }
};
std::tuple<Tensor, Tensor> policy_loss(const Tensor& logits_, const Tensor& ids_, const OptTensor& old_logp, const Tensor& advantages, const OptTensor& mask_, const OptTensor& ref_logp,
                                       double low, double high, double kl, double denom) {
    Tensor logits = logits_, ids = ids_, mask = given(mask_);
    check_plain("policy_loss", logits_, ids_, given(mask_), given(old_logp), advantages, given(ref_logp));
    check_rows("policy_loss", logits, ids, mask);
    const PolicyArgs a = policy_args(logits, ids, old_logp, advantages, ref_logp, low, high, kl, denom);
    if (needs_grad(logits)) {
        const variable_list y = PolicyLoss::apply(logits, Plain{ids}, Plain{mask}, a);
        return {y[0], y[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, logp] = policy_forward(logits, ids, mask, a, nullptr, nullptr);
    return {loss, logp};
}
std::tuple<Tensor, Tensor, Tensor> policy_loss_grad(const Tensor& logits_, const Tensor& ids_, const OptTensor& old_logp, const Tensor& advantages, const OptTensor& mask_,
                                                    const OptTensor& ref_logp, double low, double high, double kl, double denom, double scale, const OptTensor& out_) {
    Tensor logits = logits_, ids = ids_, mask = given(mask_), out = given(out_);
    check_plain("policy_loss_grad", logits_, ids_, given(mask_), given(old_logp), advantages, given(ref_logp), given(out_));
    check_rows("policy_loss_grad", logits, ids, mask);
    const PolicyArgs a = policy_args(logits, ids, old_logp, advantages, ref_logp, low, high, kl, denom);
    // (torch refuses its own operators in place over these; a tensor that is no leaf has its version counted up)
    const bool over_leaf = needs_grad(out) && (out.is_leaf() || (out.is_view() && out._base().is_leaf()));
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(logits.device());
    if (!out.defined()) out = like(logits.sizes(), logits, logits.scalar_type());
    TORCH_CHECK(out.sizes() == logits.sizes() && out.scalar_type() == logits.scalar_type() && out.device() == logits.device() && out.is_contiguous(),
                "policy_loss_grad: out must be dense and like the logits");
    if (out_.has_value()) {
        TORCH_CHECK(!over_leaf, "policy_loss_grad: out is a leaf that requires a gradient, or a view of one");
        at::assert_no_partial_overlap(out, logits_);
        if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();   // written in place: what autograd has kept of it is no longer good
    }
    const Rows r(logits, ids, mask);
    Tensor loss = like({}, logits, at::kFloat), logp = like(ids.sizes(), logits, at::kFloat), scratch = like({r.t.rows + 1}, logits, at::kDouble);
    check(lib.ab_policy_loss_grad(&r.t, &a.p, (float)scale, f32(loss), f32(logp), out.data_ptr(), scratch.data_ptr<double>(), stream()), "ab_policy_loss_grad");
    return {loss, logp, out};
}

std::pair<Tensor, Tensor> preference_forward(const Tensor& logits, const Tensor& ids, const Tensor& mask, const Tensor& ref, double beta, double smoothing, Tensor* stats, Tensor* g) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const Rows r(logits, ids, mask);
    const int64_t n = ids.size(0), T = ids.size(1);
    Tensor loss = like({}, logits, at::kFloat), logp = like({n}, logits, at::kFloat), scratch = like({n * T}, logits, at::kDouble);
    if (stats) *stats = like({n * T, 2}, logits, at::kFloat), *g = like({n}, logits, at::kFloat);
    check(lib.ab_preference_loss_fwd(&r.t, n / 2, T, f32(ref), (float)beta, (float)smoothing, f32(loss), f32(logp), stats ? f32(*stats) : nullptr, stats ? f32(*g) : nullptr,
                                     scratch.data_ptr<double>(), stream()), "ab_preference_loss_fwd");
    return {loss, logp};
}
struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
    static variable_list forward(AutogradContext* ctx, Tensor logits, Plain ids_, Plain mask_, Plain ref, double beta, double smoothing) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &ids = ids_.t, &mask = mask_.t;
        Tensor stats, g;
        auto [loss, logp] = preference_forward(logits, ids, mask, ref.t, beta, smoothing, &stats, &g);
        ctx->save_for_backward({logits, ids, mask, stats, g});
        ctx->mark_non_differentiable({logp});
        return {loss, logp};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward(grads);
        const variable_list s = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        variable_list out(6);
        out[0] = dlogits_of(s[0], s[1], s[2], s[3], s[4], std::max<int64_t>(1, s[1].size(1)), grads[0].contiguous());
        return out;
    }
};
std::tuple<Tensor, Tensor> preference_loss(const Tensor& logits_, const Tensor& ids_, const Tensor& ref_logp, const OptTensor& mask_, double beta, double smoothing) {
    Tensor logits = logits_, ids = ids_, mask = given(mask_);
    check_plain("preference_loss", logits_, ids_, given(mask_), ref_logp);
    check_rows("preference_loss", logits, ids, mask);
    TORCH_CHECK(logits.dim() == 3 && logits.size(0) % 2 == 0 && logits.size(0) > 0, "preference_loss: logits must be [2 P, T, V]");
    TORCH_CHECK(ref_logp.sizes() == at::IntArrayRef({logits.size(0)}) && ref_logp.device() == logits.device(), "preference_loss: ref_logp must be [2 P] on the device of logits");
    TORCH_CHECK(smoothing >= 0 && smoothing <= 1, "preference_loss: label_smoothing outside 0 .. 1");
    const Tensor ref = ref_logp.detach().to(at::kFloat).contiguous();
    if (needs_grad(logits)) {
        const variable_list y = PreferenceLoss::apply(logits, Plain{ids}, Plain{mask}, Plain{ref}, beta, smoothing);
        return {y[0], y[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, logp] = preference_forward(logits, ids, mask, ref, beta, smoothing, nullptr, nullptr);
    return {loss, logp};
}

// ---- the norm over all gradients -------------------------------------------------------------------------------------------------------
bool same_order(const Tensor& a, const Tensor& b) { return a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous()); }
// out: empty (the norm alone), the gradients themselves, or one tensor for each. What is not dense, or lies in another order than its
// gradient, goes by way of a copy.
Tensor clip_grad_norm(at::TensorList grads, double max_norm, double scale, at::TensorList out) {
    constexpr const char* who = "clip_grad_norm";
    TORCH_CHECK(!grads.empty(), who, ": no gradients");
    TORCH_CHECK(out.empty() || out.size() == grads.size(), who, ": ", std::to_string(grads.size()), " gradients and ", std::to_string(out.size()), " outputs");
    TORCH_CHECK(scale > 0 && scale <= std::numeric_limits<float>::max(), who, ": the scale must be positive and finite, in 32 bits");
    TORCH_CHECK(max_norm >= 0, who, ": the largest norm is negative or not a number");
    check_plain(who);
    const at::Device device = grads[0].device();
    const bool grad_mode = at::GradMode::is_enabled();
    std::vector<ab_grad> list(grads.size());
    std::vector<Tensor> copies;                         // kept until the kernels are launched
    std::vector<std::pair<size_t, Tensor>> back;        // outputs that are copied to where they belong
    auto fits = [&](const Tensor& t) {   // (what has no autograd metadata has no tangent)
        return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.device() == device && is_known(t) && t.has_storage() && !t.is_neg() &&
               (!t.unsafeGetTensorImpl()->autograd_meta() || !t._fw_grad(/*level=*/0).defined());
    };
    at::AutoDispatchBelowADInplaceOrView below;
    for (size_t i = 0; i < grads.size(); ++i) {   // (a model has hundreds of them: what each needs is kept short)
        const Tensor& g = grads[i];
        TORCH_CHECK(fits(g), who, ": gradient ", std::to_string(i), " is not a dense fp16, bf16 or fp32 tensor on the device of the first");
        ab_grad& e = list[i];
        e = {g.data_ptr(), nullptr, g.numel(), type_of(g), AB_DT_F16};
        const bool dense = g.is_non_overlapping_and_dense();
        if (out.empty()) {
            if (!dense) e.g = copies.emplace_back(g.contiguous()).data_ptr();
            continue;
        }
        const Tensor& o = out[i];
        const bool in_place = o.is_same(g);
        TORCH_CHECK(in_place || (fits(o) && o.sizes() == g.sizes()), who, ": output ", std::to_string(i), " is not a dense fp16, bf16 or fp32 tensor of its gradient's shape and device");
        TORCH_CHECK(!(grad_mode && o.requires_grad()), who, ": output ", std::to_string(i), " requires a gradient; write over it under torch.no_grad()");
        if (dense && (in_place || (o.is_non_overlapping_and_dense() && same_order(g, o)))) {
            e.out = o.data_ptr();
        } else {
            at::assert_no_internal_overlap(o);
            e.g = copies.emplace_back(g.contiguous()).data_ptr();
            if (!in_place && o.is_contiguous()) e.out = o.data_ptr();
            else e.out = back.emplace_back(i, at::empty(g.sizes(), o.options())).second.data_ptr();
        }
        e.out_dtype = type_of(o);
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    }
    if (!back.empty()) {   // an output that is copied to its place must not lie among the values of another one: which of the two would stay?
        std::vector<std::array<uintptr_t, 3>> spans;
        for (size_t i = 0; i < out.size(); ++i) {
            if (out[i].numel() == 0) continue;
            int64_t last = 0;
            for (int64_t d = 0; d < out[i].dim(); ++d) last += (out[i].size(d) - 1) * out[i].stride(d);
            const uintptr_t at = reinterpret_cast<uintptr_t>(out[i].data_ptr());
            spans.push_back({at, at + (uintptr_t)(last + 1) * out[i].element_size(), i});
        }
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i) {
            TORCH_CHECK(spans[i][0] >= spans[i - 1][1], who, ": outputs ", std::to_string(spans[i - 1][2]), " and ", std::to_string(spans[i][2]), " lie between each other's values");
        }
    }
    const c10::cuda::CUDAGuard guard(device);
    Tensor norm = like({}, grads[0], at::kFloat), scratch = like({(int64_t)lib.ab_clip_grad_norm_scratch_bytes((int64_t)list.size())}, grads[0], at::kByte);
    check(lib.ab_clip_grad_norm(list.data(), (int64_t)list.size(), scale, max_norm, f32(norm), scratch.data_ptr(), stream()), "ab_clip_grad_norm");
    for (const auto& b : back) out[b.first].copy_(b.second);
    return norm;
}

}  // namespace

TORCH_LIBRARY(albatross_b200, m) {
    m.def("wkv7(Tensor? state, Tensor r, Tensor w, Tensor k, Tensor v, Tensor a, Tensor b, Tensor? lengths) -> (Tensor, Tensor)", wkv7);
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, int groups) -> Tensor", layer_norm);
    m.def("token_logp(Tensor logits, Tensor ids, Tensor? mask) -> Tensor", token_logp);
    m.def("policy_loss(Tensor logits, Tensor ids, Tensor? old_logp, Tensor advantages, Tensor? mask, Tensor? ref_logp, float clip_low, float clip_high, float kl, float denom) "
          "-> (Tensor, Tensor)", policy_loss);
    m.def("policy_loss_grad(Tensor logits, Tensor ids, Tensor? old_logp, Tensor advantages, Tensor? mask, Tensor? ref_logp, float clip_low, float clip_high, float kl, float denom, "
          "float scale, Tensor? out) -> (Tensor, Tensor, Tensor)", policy_loss_grad);
    m.def("preference_loss(Tensor logits, Tensor ids, Tensor ref_logp, Tensor? mask, float beta, float smoothing) -> (Tensor, Tensor)", preference_loss);
}

// clip_grad_norm for lists of hundreds of tensors: the dispatcher boxes and unboxes both lists, 0.2 us a tensor of the 0.3 that a call
// takes. Takes Python lists or tuples of tensors (out: None, for the norm alone) with the interpreter's lock held; returns null, with the
// error set, where it throws. Neither dispatch modes nor the profiler see the call.
struct LetGo {   // of the interpreter's lock: a launch may have to wait for room in the queue, and what it waits for may need that lock (a host function)
    PyThreadState* const state = PyEval_SaveThread();
    LetGo() = default;
    LetGo(const LetGo&) = delete;
    ~LetGo() { PyEval_RestoreThread(state); }
};
static bool tensors_of(PyObject* list, std::vector<Tensor>& out) {
    PyObject* fast = PySequence_Fast(list, "clip_grad_norm: a list of tensors is expected");
    if (!fast) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    out.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* t = PySequence_Fast_GET_ITEM(fast, i);
        if (!THPVariable_Check(t)) {
            Py_DECREF(fast);
            PyErr_SetString(PyExc_RuntimeError, "clip_grad_norm: a list of tensors is expected");
            return false;
        }
        out.push_back(THPVariable_Unpack(t));
    }
    Py_DECREF(fast);
    return true;
}
extern "C" PyObject* albatross_b200_clip_grad_norm(PyObject* grads, double max_norm, double scale, PyObject* out) {
    try {
        std::vector<Tensor> g, o;
        if (!tensors_of(grads, g) || (out != Py_None && out != grads && !tensors_of(out, o))) return nullptr;
        Tensor norm;
        {
            const LetGo lock;
            norm = clip_grad_norm(g, max_norm, scale, out == grads ? g : o);
        }
        return THPVariable_Wrap(norm);
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());   // (as torch's own bindings do: memory that runs out is torch.OutOfMemoryError)
    }
    return nullptr;
}

// Takes the entries from the kernel library at `path` (already loaded). 0, or -1 with what is missing in `missing`.
extern "C" int albatross_b200_train_bind(const char* path, const char** missing) {
    void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    *missing = path;
    if (!h) return -1;
    AB_TAKE(ab_last_error)
    AB_TAKE(ab_wkv7_checkpoint_bytes)
    AB_TAKE(ab_wkv7_seq_fwd)
    AB_TAKE(ab_wkv7_seq_bwd)
    AB_TAKE(ab_layer_norm_fwd)
    AB_TAKE(ab_layer_norm_scratch_bytes)
    AB_TAKE(ab_layer_norm_bwd)
    AB_TAKE(ab_token_logp_fwd)
    AB_TAKE(ab_token_logp_bwd)
    AB_TAKE(ab_policy_loss_fwd)
    AB_TAKE(ab_policy_loss_grad)
    AB_TAKE(ab_preference_loss_fwd)
    AB_TAKE(ab_clip_grad_norm_scratch_bytes)
    AB_TAKE(ab_clip_grad_norm)
    last_error = lib.ab_last_error;
    return 0;
}
