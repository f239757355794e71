// What the operator shims (train_op.cpp, serve_op.cpp) share: arguments and messages.
#pragma once
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <string>

#include "../../include/albatross_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

decltype(&::ab_last_error) last_error = nullptr;   // the kernel library's, set when a shim is bound to it

// (numbers go into messages as strings: a number formatted by the stream of a shim built with another compiler's library than torch's has crashed)
void check(int status, const char* what) { TORCH_CHECK(status == AB_OK, what, " failed with status ", std::to_string(status), ": ", last_error()); }

int type_of(const Tensor& t) { return t.scalar_type() == at::kHalf ? AB_DT_F16 : t.scalar_type() == at::kBFloat16 ? AB_DT_BF16 : AB_DT_F32; }
bool is_16bit(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool is_known(const Tensor& t) { return is_16bit(t) || t.scalar_type() == at::kFloat; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
void* stream() { return (void*)at::cuda::getCurrentCUDAStream().stream(); }
Tensor like(at::IntArrayRef sizes, const Tensor& t, at::ScalarType type) { return at::empty(sizes, t.options().dtype(type)); }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
template <class... T>
bool needs_grad(const T&... t) { return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...); }
// a tensor that autograd does not look at, or none
struct Plain {
    Tensor t;
};
OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
// What would be lost without a word. A trace in the making would hold the outputs' allocation and not the call, and torch.func's wrappers have no
// memory. A tangent's tensor need not require a gradient, and would be taken below autograd.
bool traced() {
    using Key = c10::impl::TorchDispatchModeKey;
    for (const Key k : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL})
        if (c10::impl::TorchDispatchModeTLS::get_mode(k).has_value()) return true;
    return false;
}
template <class... T>
void check_plain(const char* who, const T&... t) {
    TORCH_CHECK(!traced() && ((!t.defined() || t.has_storage()) && ...), who,
                ": cannot be traced or transformed (torch.compile, torch.export, make_fx, torch.func.grad); in a compiled program call it from a function under torch.compiler.disable");
    TORCH_CHECK(!((t.defined() && t._fw_grad(/*level=*/0).defined()) || ...), who, ": forward-mode derivatives are not available");
}
// [..., C] with a dense last dimension and one stride between rows, of `least` values or more; others are copied. Here, ahead of autograd, so that
// the backward pass reads the same copy (logits[:, :-1] of several sequences are copied once, not once in each pass).
Tensor one_stride(const Tensor& t, int64_t least) {
    bool fits = t.dim() < 1 || t.size(-1) <= 1 || t.stride(-1) == 1;
    int64_t outer = -1;   // the stride that goes with the dimensions so far
    for (int64_t d = t.dim() - 2; d >= 0 && fits; --d) {
        if (t.size(d) == 1) continue;
        fits = outer < 0 ? t.stride(d) >= least : t.stride(d) == outer;
        outer = t.stride(d) * t.size(d);
    }
    return fits || t.numel() == 0 ? t : t.contiguous();
}
// [..., C] as rows [n, C] with a dense last dimension; a view where the strides allow one
Tensor as_rows(const Tensor& t) {
    const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return r.stride(1) == 1 || r.size(1) <= 1 ? r : r.contiguous();
}

}  // namespace

// Takes an entry from the kernel library `h`; what is missing goes to `missing`.
#define AB_TAKE(name)                                                                         \
    lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(h, #name));                         \
    if (!lib.name) {                                                                          \
        *missing = #name;                                                                     \
        return -1;                                                                            \
    }
