// What the sources of the torch ops share: the checks of a tensor argument, the error of a failed call of the C library,
// the device and stream of a call.
#ifndef OEQ_TORCH_H
#define OEQ_TORCH_H

#include "oeq_amd.h"

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <optional>
#include <string>

namespace oeq_torch {

using at::Tensor;

// Throws the package's Python exception (oeq_torch.cpp).
[[noreturn]] void raise(const std::string& text);

inline void check(int rc, const char* what) {
    if (rc == OEQ_OK) return;
    const char* msg = oeq_last_error();
    raise(std::string(what) + " failed (" + std::to_string(rc) + "): " + (msg ? msg : ""));
}

inline int dtype_code(at::ScalarType t) {  // the reference's codes
    switch (t) {
        case at::kFloat: return 1;
        case at::kDouble: return 2;
        case at::kInt: return 3;
        case at::kLong: return 4;
        case at::kByte: return 5;
        default: return 0;
    }
}

inline std::string dtype_text(at::ScalarType t) {
    const int code = dtype_code(t);
    return code ? std::to_string(code) : std::string(at::toString(t));
}

// `beside`: another operand of the call, on whose device all of them have to be (a kernel would read another device's
// memory through a pointer that need not mean anything on its own).
inline void check_tensor(const Tensor& t, at::IntArrayRef shape, at::ScalarType dtype, const char* name, const Tensor& beside) {
    TORCH_CHECK(t.sizes() == shape, "Shape mismatch for tensor '", name, "'. Expected: ", shape, ". Got: ", t.sizes());
    TORCH_CHECK(t.is_cuda(), "Tensor '", name, "' is not on the GPU.");
    TORCH_CHECK(t.device() == beside.device(), "Tensor '", name, "' is on ", t.device(), ", not on ", beside.device(),
                " as the operands before it.");
    TORCH_CHECK(t.scalar_type() == dtype, "Dtype mismatch for tensor '", name, "'. Expected: ", dtype_text(dtype),
                ". Got: ", dtype_text(t.scalar_type()));
}

// The device of a call's operands made current, and torch's stream on it.
struct OnDevice {
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
    void* stream;
    explicit OnDevice(const Tensor& t) : guard(t.device()) {
        stream = (void*)(hipStream_t)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index());
    }
};

inline Tensor scratch(const Tensor& like, size_t bytes) {
    return at::empty({(int64_t)(bytes ? bytes : 1)}, like.options().dtype(at::kByte));
}

using OptTensor = std::optional<Tensor>;

inline bool wants_grad(const Tensor& t) { return t.requires_grad(); }
inline bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
inline Tensor tangent_of(const Tensor& t) { return t.defined() ? Tensor(t._fw_grad(0)) : Tensor(); }
inline Tensor tangent_of(const OptTensor& t) { return t.has_value() ? tangent_of(*t) : Tensor(); }

// Whether a call of differentiable operands is recorded for a backward pass.
template <typename... Ts>
bool records(const Ts&... ts) {
    return at::GradMode::is_enabled() && (wants_grad(ts) || ...);
}

// Whether an operand is a dual tensor of forward-mode differentiation. Such a tensor need not require a gradient: below
// autograd its tangent would be lost and the derivative come out as zero.
template <typename... Ts>
bool has_tangent(const Ts&... ts) {
    return (tangent_of(ts).defined() || ...);
}
template <typename... Ts>
void refuse_tangents(const char* op, const Ts&... ts) {
    TORCH_CHECK(!has_tangent(ts...), op, " has no forward-mode derivative: differentiate it backward");
}

}  // namespace oeq_torch
#endif
