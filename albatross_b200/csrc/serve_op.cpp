// What serves a token, as torch operators beside those of train_op.cpp (torch.ops.albatross_b200.*): arguments checked, memory from torch's
// allocator, the C entries called on torch's current stream of the tensors' device. Neither has gradients.
#include "op.h"

namespace {

struct Entries {
#define AB_ENTRY(name) decltype(&::name) name = nullptr
    AB_ENTRY(ab_last_error);
    AB_ENTRY(ab_sample_filtered);
    AB_ENTRY(ab_linear_int4);
#undef AB_ENTRY
} lib;

// one number per row, dense on the device; `type`: what it is read as
const Tensor per_row(const char* what, const OptTensor& t, const Tensor& logits, int64_t rows, at::ScalarType type) {
    if (!t.has_value()) return Tensor();
    check_plain("sampler_batch", *t);
    TORCH_CHECK(t->device() == logits.device() && t->numel() == rows && (type == at::kInt ? at::isIntegralType(t->scalar_type(), false) && t->scalar_type() != at::kUInt64 : at::isFloatingType(t->scalar_type())),
                "sampler_batch: ", what, " must be a number, or a tensor of one ", type == at::kInt ? "whole" : "floating", " number per row on the device of logits");
    // (a k that 32 bits do not hold filters nothing)
    return (type == at::kInt && t->scalar_type() == at::kLong ? t->clamp(INT32_MIN, INT32_MAX) : *t).to(type).contiguous();
}
// whether the bytes [from, to) meet one of n runs of `length` bytes that begin `step` apart
bool meets(uintptr_t from, uintptr_t to, const void* base_, uint64_t n, uint64_t length, uint64_t step) {
    const uintptr_t base = reinterpret_cast<uintptr_t>(base_);
    if (from == to || n == 0 || length == 0) return false;
    const uint64_t ended = from < base + length ? 0 : step == 0 ? n : (from - base - length) / step + 1;   // runs that end in front of it
    return ended < n && base + ended * step < to;
}
bool meets(uintptr_t from, uintptr_t to, const Tensor& dense) { return dense.defined() && meets(from, to, dense.data_ptr(), 1, dense.nbytes(), 0); }
std::tuple<Tensor, Tensor> sample(const Tensor& logits_, const Tensor& uniform, const OptTensor& temperature, const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p,
                                  double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all, const OptTensor& out_) {
    constexpr const char* who = "sampler_batch";
    check_plain(who, logits_, uniform, given(out_));
    TORCH_CHECK(logits_.is_cuda() && is_known(logits_) && logits_.dim() >= 1 && logits_.size(-1) > 0 && logits_.size(-1) <= 1 << 18, who,
                ": logits must be [..., V], fp16, bf16 or fp32, on a CUDA device, with V up to 2^18");
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(logits_.device());
    const Tensor rows = as_rows(one_stride(logits_, 0));
    const int64_t n = rows.size(0), V = rows.size(1);
    TORCH_CHECK(uniform.scalar_type() == at::kFloat && uniform.numel() == n && uniform.device() == rows.device(), who, ": uniform must be fp32, one number per row, on the device of logits");
    const Tensor u = uniform.contiguous(), T = per_row("temperature", temperature, rows, n, at::kFloat), p = per_row("top_p", top_p, rows, n, at::kFloat),
                 m = per_row("min_p", min_p, rows, n, at::kFloat), k = per_row("top_k", top_k, rows, n, at::kInt);
    at::DimVector sizes(logits_.sizes().begin(), logits_.sizes().end());
    sizes.back() = 1;
    Tensor ids = given(out_), logp = like(sizes, rows, at::kFloat);
    if (ids.defined()) {
        TORCH_CHECK(ids.scalar_type() == at::kLong && ids.numel() == n && ids.is_contiguous() && (ids.device() == rows.device() || (ids.is_cpu() && ids.is_pinned())), who,
                    ": out must be a dense int64 tensor of one id per row, on the device of logits or in pinned host memory");
        // (rows are drawn side by side: an id must not fall into what another row still reads)
        const uintptr_t from = reinterpret_cast<uintptr_t>(ids.data_ptr()), to = from + ids.nbytes();
        TORCH_CHECK(!(ids.is_cuda() && (meets(from, to, rows.data_ptr(), n, V * rows.element_size(), rows.stride(0) * rows.element_size()) || meets(from, to, u) || meets(from, to, T) ||
                                        meets(from, to, p) || meets(from, to, m) || meets(from, to, k))),
                    who, ": out lies among the values of an input");
        if (!ids.is_inference()) ids.unsafeGetTensorImpl()->bump_version();
    } else {
        ids = like(sizes, rows, at::kLong);
    }
    const ab_sampling s = {f32(T), f32(p), f32(m), k.defined() ? k.data_ptr<int32_t>() : nullptr, temperature_all, top_p_all, min_p_all,
                           (int32_t)std::max<int64_t>(0, std::min<int64_t>(top_k_all, INT32_MAX)), 0};
    check(lib.ab_sample_filtered(type_of(rows), n, (int)V, ptr(rows), rows.stride(0), f32(u), &s, ids.data_ptr<int64_t>(), f32(logp), stream()), "ab_sample_filtered");
    return {out_.has_value() ? ids.view(sizes) : ids, logp};
}

Tensor linear_int4(const Tensor& x_, const Tensor& w, const Tensor& scale, const OptTensor& zero_) {
    constexpr const char* who = "linear_int4";
    const Tensor zero = given(zero_);
    check_plain(who, x_, w, scale, zero);
    TORCH_CHECK(x_.is_cuda() && is_16bit(x_) && x_.dim() >= 1, who, ": x must be [..., K], fp16 or bf16, on a CUDA device");
    TORCH_CHECK(!needs_grad(x_, scale), who, ": has no gradients; call it under torch.no_grad()");
    const int64_t K = x_.size(-1);
    TORCH_CHECK(w.dim() == 2 && w.scalar_type() == at::kByte && w.device() == x_.device() && w.size(0) > 0 && w.size(0) <= INT32_MAX && K > 0 && K <= INT32_MAX && 2 * w.size(1) == K, who,
                ": w must be uint8 [N, K / 2] on the device of x, two codes a byte");
    const int64_t N = w.size(0);
    TORCH_CHECK(scale.dim() == 2 && scale.scalar_type() == x_.scalar_type() && scale.device() == x_.device() && scale.size(0) == N && scale.size(1) > 0 && K % scale.size(1) == 0, who,
                ": scale must be [N, K / group] of the type and device of x");
    TORCH_CHECK(!zero.defined() || (zero.scalar_type() == at::kByte && zero.device() == x_.device() && zero.sizes() == scale.sizes()), who, ": zero must be uint8, of the shape and device of scale");
    TORCH_CHECK(w.is_contiguous() && scale.is_contiguous() && (!zero.defined() || zero.is_contiguous()), who, ": w, scale and zero must be dense (lay them out once, not in every call)");
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = as_rows(one_stride(x_, 0));
    TORCH_CHECK(x.size(0) <= INT32_MAX, who, ": too many rows");
    at::DimVector sizes(x_.sizes().begin(), x_.sizes().end());
    sizes.back() = N;
    Tensor y = like(sizes, x, x.scalar_type());
    const ab_int4 m = {type_of(x), (int32_t)N, (int32_t)K, (int32_t)(K / scale.size(1)), w.data_ptr(), scale.data_ptr(), ptr(zero)};
    check(lib.ab_linear_int4(&m, (int)x.size(0), ptr(x), x.stride(0), ptr(y), stream()), "ab_linear_int4");
    return y;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(albatross_b200, m) {
    m.def("sample(Tensor logits, Tensor uniform, Tensor? temperature, Tensor? top_k, Tensor? top_p, Tensor? min_p, float temperature_all, int top_k_all, float top_p_all, "
          "float min_p_all, Tensor? out) -> (Tensor, Tensor)", sample);
    m.def("linear_int4(Tensor x, Tensor w, Tensor scale, Tensor? zero) -> Tensor", linear_int4);
}

// Takes the entries from the kernel library at `path` (already loaded). 0, or -1 with what is missing in `missing`.
extern "C" int albatross_b200_serve_bind(const char* path, const char** missing) {
    void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    *missing = path;
    if (!h) return -1;
    AB_TAKE(ab_last_error)
    AB_TAKE(ab_sample_filtered)
    AB_TAKE(ab_linear_int4)
    last_error = lib.ab_last_error;
    return 0;
}
