// The torch ops of the operators on the nodes of a batch: checks, allocation, launches through the C ABI and autograd.
// (Schemas and fake kernels: _torch/nodes.py.) The first derivatives of attention and of the norm with rotation are ops of
// their own, whose derivatives are refused; the gradient of dropout is dropout of the gradient, to any order.
#include "oeq_torch.h"

#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

using namespace oeq_torch;
using Tensor2 = std::tuple<Tensor, Tensor>;
using Tensor3 = std::tuple<Tensor, Tensor, Tensor>;
using Tensor4 = std::tuple<Tensor, Tensor, Tensor, Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

int element_of(const Tensor& t, const char* name, bool wide = false) {
    switch (t.scalar_type()) {
        case at::kFloat: return OEQ_FLOAT32;
        case at::kHalf: return OEQ_FLOAT16;
        case at::kBFloat16: return OEQ_BFLOAT16;
        case at::kDouble:
            if (wide) return OEQ_FLOAT64;
        default:
            TORCH_CHECK(false, "Dtype mismatch for tensor '", name, "'. Expected: float32, float16", wide ? ", bfloat16 or float64" : " or bfloat16",
                        ". Got: ", at::toString(t.scalar_type()));
    }
}

void check_heads(const Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() == 3, "Shape mismatch for tensor '", name, "'. Expected: [rows, heads, head_dim]. Got: ", t.sizes());
}

// Rows of heads as the kernels take them: a head's elements one after the other, everything at multiples of 16 bytes, a row
// not too far from the next for 32-bit offsets within a tile. A view that is like this (queries, keys and values of one
// projection, say) is read in place.
struct Rows {
    Tensor t;
    int64_t row = 0, head = 0;
    Rows() = default;
    explicit Rows(const Tensor& x) : t(x) {
        if (!fits(t)) t = x.contiguous();
        if (!fits(t)) t = x.clone(at::MemoryFormat::Contiguous);
        row = t.size(0) > 1 ? t.stride(0) : 0;
        head = t.size(1) > 1 ? t.stride(1) : 0;
    }
    static bool fits(const Tensor& t) {
        const int64_t bytes = t.element_size();
        const auto far = [&](int dim) { return t.size(dim) > 1 ? t.stride(dim) * bytes : 0; };
        return (t.size(2) <= 1 || t.stride(2) == 1) && far(0) % 16 == 0 && far(1) % 16 == 0 && far(0) >= 0 && far(1) >= 0 &&
               far(0) < (1 << 24) && ((uintptr_t)t.data_ptr() & 15) == 0;
    }
};

Tensor whole(const Tensor& t) {  // contiguous, from a multiple of 16 bytes on
    const Tensor c = t.contiguous();
    return (uintptr_t)c.data_ptr() & 15 ? c.clone() : c;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

struct Attention {
    oeq_attention a{};
    Rows q, k, v;
    Tensor q_ptr, k_ptr, k_len;

    Attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& q_ptr_, const Tensor& k_ptr_,
              const OptTensor& k_len_, bool causal, double scale) {
        check_heads(q_, "q");
        a.type = element_of(q_, "q");
        const int64_t d = q_.size(2);
        TORCH_CHECK(d > 0 && d <= 128 && d % 8 == 0, "Shape mismatch for tensor 'q'. Expected: head_dim a multiple of 8 up to ",
                    "128. Got: ", q_.sizes());
        check_heads(k_, "k");
        check_tensor(q_, q_.sizes(), q_.scalar_type(), "q", q_);
        check_tensor(k_, {k_.size(0), k_.size(1), d}, q_.scalar_type(), "k", q_);
        check_tensor(v_, k_.sizes(), q_.scalar_type(), "v", q_);
        TORCH_CHECK(q_.size(1) > 0 && k_.size(1) > 0 && q_.size(1) % k_.size(1) == 0,
                    "Shape mismatch for tensor 'k'. Expected: a number of heads that divides the ", q_.size(1),
                    " heads of 'q'. Got: ", k_.sizes());
        TORCH_CHECK(q_ptr_.dim() == 1 && q_ptr_.size(0) > 0,
                    "Shape mismatch for tensor 'q_ptr'. Expected: [segments + 1]. Got: ", q_ptr_.sizes());
        check_tensor(q_ptr_, q_ptr_.sizes(), at::kLong, "q_ptr", q_);
        check_tensor(k_ptr_, q_ptr_.sizes(), at::kLong, "k_ptr", q_);
        if (k_len_.has_value()) check_tensor(*k_len_, {q_ptr_.size(0) - 1}, at::kLong, "k_len", q_);
        TORCH_CHECK(scale > 0 && std::isfinite(scale), "packed_attention: scale must be positive, got ", scale);
        q = Rows(q_), k = Rows(k_), v = Rows(v_);
        q_ptr = q_ptr_.contiguous(), k_ptr = k_ptr_.contiguous();
        if (k_len_.has_value()) k_len = k_len_->contiguous();
        a.causal = causal;
        a.segments = (int32_t)(q_ptr.size(0) - 1);
        a.q_heads = (int32_t)q_.size(1), a.k_heads = (int32_t)k_.size(1), a.head_dim = (int32_t)d;
        a.scale = (float)scale;
        a.q_rows = q_.size(0), a.k_rows = k_.size(0);
        a.q_row_stride = q.row, a.q_head_stride = q.head;
        a.k_row_stride = k.row, a.k_head_stride = k.head;
        a.v_row_stride = v.row, a.v_head_stride = v.head;
        a.q = q.t.data_ptr(), a.k = k.t.data_ptr(), a.v = v.t.data_ptr();
        a.q_ptr = q_ptr.data_ptr<int64_t>(), a.k_ptr = k_ptr.data_ptr<int64_t>();
        a.k_len = k_len.defined() ? k_len.data_ptr<int64_t>() : nullptr;
    }
};

// (out, log2_sum, rest): `rest`, what rounding took off `out`, is kept for a pass that will be differentiated, where the
// type has 16 bits; else it is empty.
Tensor3 packed_attention_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr, const Tensor& k_ptr,
                             const OptTensor& k_len, bool causal, double scale, bool keep_rest) {
    const Attention call(q, k, v, q_ptr, k_ptr, k_len, causal, scale);
    OnDevice dev(q);
    Tensor out = at::empty(q.sizes(), q.options());
    Tensor log2_sum = at::empty({q.size(1), oeq_attention_stat_stride(q.size(0))}, q.options().dtype(at::kFloat));
    keep_rest = keep_rest && q.element_size() == 2;
    Tensor rest = keep_rest ? at::empty(q.sizes(), q.options()) : at::empty({0}, q.options());
    const size_t nb = oeq_attention_forward_workspace_bytes(&call.a);
    Tensor ws;
    if (nb) ws = scratch(q, nb);
    check(oeq_attention_forward(&call.a, out.data_ptr(), keep_rest ? rest.data_ptr() : nullptr, log2_sum.data_ptr<float>(),
                                nb ? ws.data_ptr() : nullptr, nb, dev.stream),
          "oeq_attention_forward");
    return {out, log2_sum, rest};
}

Tensor3 packed_attention_backward_gpu(const Tensor& grad, const Tensor& q, const Tensor& k, const Tensor& v,
                                      const Tensor& out, const Tensor& log2_sum, const Tensor& rest, const Tensor& q_ptr,
                                      const Tensor& k_ptr, const OptTensor& k_len, bool causal, double scale) {
    check_heads(q, "q");
    check_tensor(grad, q.sizes(), q.scalar_type(), "grad", q);
    check_tensor(out, q.sizes(), q.scalar_type(), "out", q);
    check_tensor(log2_sum, {q.size(1), oeq_attention_stat_stride(q.size(0))}, at::kFloat, "log2_sum", q);
    if (rest.numel()) check_tensor(rest, q.sizes(), q.scalar_type(), "rest", q);
    const Attention call(q, k, v, q_ptr, k_ptr, k_len, causal, scale);
    OnDevice dev(q);
    const Rows g(grad);
    const Tensor o = whole(out), sums = log2_sum.contiguous(), r = whole(rest);
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
    const size_t nb = oeq_attention_backward_workspace_bytes(&call.a);
    const Tensor ws = scratch(q, nb);
    check(oeq_attention_backward(&call.a, o.data_ptr(), r.numel() ? r.data_ptr() : nullptr, sums.data_ptr<float>(),
                                 g.t.data_ptr(), g.row, g.head, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                 ws.data_ptr(), nb, dev.stream),
          "oeq_attention_backward");
    return {dq, dk, dv};
}

// ---------------------------------------------------------------------------
// norm and rotation
// ---------------------------------------------------------------------------

struct Rotary {
    oeq_qk_rotary a{};
    Rows q, k;
    Tensor positions, table, q_weight, k_weight;

    Rotary(const Tensor& q_, const Tensor& k_, const Tensor& positions_, const Tensor& table_, const OptTensor& q_weight_,
           const OptTensor& k_weight_, double eps, bool interleaved) {
        check_heads(q_, "q");
        a.type = element_of(q_, "q");
        const int64_t n = q_.size(0), d = q_.size(2);
        TORCH_CHECK(d > 0 && d <= 128 && d % 8 == 0, "Shape mismatch for tensor 'q'. Expected: head_dim a multiple of 8 up to ",
                    "128. Got: ", q_.sizes());
        check_heads(k_, "k");
        check_tensor(q_, q_.sizes(), q_.scalar_type(), "q", q_);
        check_tensor(k_, {n, k_.size(1), d}, q_.scalar_type(), "k", q_);
        check_tensor(positions_, {n}, at::kLong, "positions", q_);
        TORCH_CHECK(table_.dim() == 3 && table_.size(1) == 2 && table_.size(2) % 4 == 0 && 2 * table_.size(2) <= d,
                    "Shape mismatch for tensor 'table'. Expected: [positions, 2, rotary_dim / 2] with rotary_dim a multiple ",
                    "of 8 up to ", d, ". Got: ", table_.sizes());
        check_tensor(table_, table_.sizes(), at::kFloat, "table", q_);
        if (q_weight_.has_value()) check_tensor(*q_weight_, {d}, q_.scalar_type(), "q_weight", q_);
        if (k_weight_.has_value()) check_tensor(*k_weight_, {d}, q_.scalar_type(), "k_weight", q_);
        TORCH_CHECK(eps >= 0, "qk_norm_rotary: eps must not be negative, got ", eps);
        q = Rows(q_), k = Rows(k_);
        positions = positions_.contiguous(), table = whole(table_);
        if (q_weight_.has_value()) q_weight = whole(*q_weight_), a.q_weight = q_weight.data_ptr();
        if (k_weight_.has_value()) k_weight = whole(*k_weight_), a.k_weight = k_weight.data_ptr();
        a.interleaved = interleaved;
        a.q_heads = (int32_t)q_.size(1), a.k_heads = (int32_t)k_.size(1), a.head_dim = (int32_t)d;
        a.rotary_dim = (int32_t)(2 * table.size(2));
        a.eps = (float)eps;
        a.rows = n, a.table_rows = table.size(0);
        a.q_row_stride = q.row, a.q_head_stride = q.head;
        a.k_row_stride = k.row, a.k_head_stride = k.head;
        a.q = q.t.data_ptr(), a.k = k.t.data_ptr();
        a.positions = positions.data_ptr<int64_t>(), a.table = table.data_ptr<float>();
    }
};

Tensor2 qk_norm_rotary_gpu(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& table,
                           const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved) {
    const Rotary call(q, k, positions, table, q_weight, k_weight, eps, interleaved);
    OnDevice dev(q);
    Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
    check(oeq_qk_norm_rotary(&call.a, q_out.data_ptr(), k_out.data_ptr(), dev.stream), "oeq_qk_norm_rotary");
    return {q_out, k_out};
}

// (the gradient of a weight that is not there is an empty tensor)
Tensor4 qk_norm_rotary_backward_gpu(const Tensor& q_grad, const Tensor& k_grad, const Tensor& q, const Tensor& k,
                                    const Tensor& positions, const Tensor& table, const OptTensor& q_weight,
                                    const OptTensor& k_weight, double eps, bool interleaved) {
    check_tensor(q_grad, q.sizes(), q.scalar_type(), "q_grad", q);
    check_tensor(k_grad, k.sizes(), q.scalar_type(), "k_grad", q);
    const Rotary call(q, k, positions, table, q_weight, k_weight, eps, interleaved);
    OnDevice dev(q);
    const Rows gq(q_grad), gk(k_grad);
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    Tensor dqw = at::empty({q_weight.has_value() ? q.size(2) : 0}, q.options());
    Tensor dkw = at::empty({k_weight.has_value() ? q.size(2) : 0}, q.options());
    const size_t nb = oeq_qk_norm_rotary_backward_workspace_bytes(&call.a);
    Tensor ws;
    if (nb) ws = scratch(q, nb);
    check(oeq_qk_norm_rotary_backward(&call.a, gq.t.data_ptr(), gq.row, gq.head, gk.t.data_ptr(), gk.row, gk.head,
                                      dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(), dkw.data_ptr(),
                                      nb ? ws.data_ptr() : nullptr, nb, dev.stream),
          "oeq_qk_norm_rotary_backward");
    return {dq, dk, dqw, dkw};
}

Tensor qk_norm_rotary_append_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions,
                                 const Tensor& table, const Tensor& k_cache, const Tensor& v_cache, const Tensor& slots,
                                 const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved) {
    check_heads(q, "q");
    check_heads(k, "k");
    check_tensor(v, k.sizes(), q.scalar_type(), "v", q);
    check_heads(k_cache, "k_cache");
    check_tensor(k_cache, {k_cache.size(0), k.size(1), k.size(2)}, q.scalar_type(), "k_cache", q);
    check_tensor(v_cache, k_cache.sizes(), q.scalar_type(), "v_cache", q);
    check_tensor(slots, {q.size(0)}, at::kLong, "slots", q);
    const Rotary call(q, k, positions, table, q_weight, k_weight, eps, interleaved);
    // the caches are written in place: a copy would not do
    TORCH_CHECK(Rows::fits(k_cache) && Rows::fits(v_cache), "qk_norm_rotary_append: the caches need heads whose elements are ",
                "contiguous and rows and heads that begin at multiples of 16 bytes");
    OnDevice dev(q);
    const Rows values(v), kc(k_cache), vc(v_cache);
    const Tensor to = slots.contiguous();
    Tensor q_out = at::empty(q.sizes(), q.options());
    check(oeq_qk_norm_rotary_append(&call.a, values.t.data_ptr(), values.row, values.head, q_out.data_ptr(), kc.t.data_ptr(),
                                    kc.row, kc.head, vc.t.data_ptr(), vc.row, vc.head, to.data_ptr<int64_t>(),
                                    k_cache.size(0), dev.stream),
          "oeq_qk_norm_rotary_append");
    return q_out;
}

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------

Tensor irrep_dropout_gpu(const Tensor& x, const OptTensor& residual, const Tensor& channels, const Tensor& seed, double p) {
    TORCH_CHECK(x.dim() == 2, "Shape mismatch for tensor 'x'. Expected: [rows, irreps.dim]. Got: ", x.sizes());
    const int type = element_of(x, "x", true);
    check_tensor(x, {x.size(0), channels.dim() == 1 ? channels.size(0) : -1}, x.scalar_type(), "x", x);
    check_tensor(channels, {x.size(1)}, at::kInt, "channels", x);
    check_tensor(seed, {2}, at::kLong, "seed", x);
    if (residual.has_value()) check_tensor(*residual, x.sizes(), x.scalar_type(), "residual", x);
    TORCH_CHECK(p >= 0 && p <= 1, "irrep_dropout: p must be between 0 and 1, got ", p);
    OnDevice dev(x);
    const Tensor in = whole(x), index = channels.contiguous(), key = seed.contiguous();
    Tensor base;
    if (residual.has_value()) base = whole(*residual);
    Tensor out = at::empty(x.sizes(), x.options());
    check(oeq_irrep_dropout(type, x.size(0), x.size(1), in.data_ptr(), base.defined() ? base.data_ptr() : nullptr,
                            out.data_ptr(), index.data_ptr<int32_t>(), key.data_ptr<int64_t>(), p, dev.stream),
          "oeq_irrep_dropout");
    return out;
}

// ---------------------------------------------------------------------------
// autograd
// ---------------------------------------------------------------------------

template <typename Sig>
auto find_op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}
#define OEQ_OP(name) \
    ([] { static const auto op = find_op<decltype(name##_gpu)>("oeq_amd::" #name); return op; }())

OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor tensor_of(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

Tensor or_zeros(const Tensor& g, const Tensor& like) { return g.defined() ? g : at::zeros_like(like); }

struct PackedAttention : public torch::autograd::Function<PackedAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr,
                                 const Tensor& k_ptr, const OptTensor& k_len, bool causal, double scale) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [out, log2_sum, rest] = OEQ_OP(packed_attention).call(q, k, v, q_ptr, k_ptr, k_len, causal, scale, true);
        ctx->save_for_backward({q, k, v, out, log2_sum, rest, q_ptr, k_ptr, tensor_of(k_len)});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({log2_sum, rest});
        return {out, log2_sum, rest};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(8);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        std::tie(out[0], out[1], out[2]) =
            OEQ_OP(packed_attention_backward)
                .call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], optional_of(s[8]), ctx->saved_data["causal"].toBool(),
                      ctx->saved_data["scale"].toDouble());
        return out;
    }
};

struct QkNormRotary : public torch::autograd::Function<QkNormRotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& positions,
                                 const Tensor& table, const OptTensor& q_weight, const OptTensor& k_weight, double eps,
                                 bool interleaved) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [q_out, k_out] = OEQ_OP(qk_norm_rotary).call(q, k, positions, table, q_weight, k_weight, eps, interleaved);
        ctx->save_for_backward({q, k, positions, table, tensor_of(q_weight), tensor_of(k_weight)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->set_materialize_grads(false);
        return {q_out, k_out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(8);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const auto s = ctx->get_saved_variables();
        auto [dq, dk, dqw, dkw] =
            OEQ_OP(qk_norm_rotary_backward)
                .call(or_zeros(grads[0], s[0]), or_zeros(grads[1], s[1]), s[0], s[1], s[2], s[3], optional_of(s[4]),
                      optional_of(s[5]), ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
        out[0] = dq, out[1] = dk;
        if (s[4].defined()) out[4] = dqw;
        if (s[5].defined()) out[5] = dkw;
        return out;
    }
};

struct IrrepDropout : public torch::autograd::Function<IrrepDropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& channels,
                          const Tensor& seed, double p) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({channels, seed});
        ctx->saved_data["p"] = p;
        ctx->saved_data["residual"] = residual.has_value();
        ctx->set_materialize_grads(false);
        return OEQ_OP(irrep_dropout).call(x, residual, channels, seed, p);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        if (ctx->needs_input_grad(0))
            out[0] = OEQ_OP(irrep_dropout).call(grads[0], OptTensor(), s[0], s[1], ctx->saved_data["p"].toDouble());
        if (ctx->saved_data["residual"].toBool()) out[1] = grads[0];
        return out;
    }
};

Tensor3 packed_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr, const Tensor& k_ptr,
                                  const OptTensor& k_len, bool causal, double scale, bool keep_rest) {
    refuse_tangents("oeq_amd::packed_attention", q, k, v);
    if (records(q, k, v)) {
        const auto out = PackedAttention::apply(q, k, v, q_ptr, k_ptr, k_len, causal, scale);
        return {out[0], out[1], out[2]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(packed_attention).call(q, k, v, q_ptr, k_ptr, k_len, causal, scale, keep_rest);
}

struct PackedAttentionGradient : public torch::autograd::Function<PackedAttentionGradient> {
    static variable_list forward(AutogradContext* ctx, const Tensor& grad, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& out, const Tensor& log2_sum, const Tensor& rest, const Tensor& q_ptr,
                                 const Tensor& k_ptr, const OptTensor& k_len, bool causal, double scale) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->set_materialize_grads(false);
        auto [dq, dk, dv] =
            OEQ_OP(packed_attention_backward).call(grad, q, k, v, out, log2_sum, rest, q_ptr, k_ptr, k_len, causal, scale);
        return {dq, dk, dv};
    }
    static variable_list backward(AutogradContext*, variable_list) {
        TORCH_CHECK(false, "Trying to backward through oeq_amd::packed_attention_backward but no autograd formula was registered.");
    }
};

Tensor3 packed_attention_backward_autograd(const Tensor& grad, const Tensor& q, const Tensor& k, const Tensor& v,
                                           const Tensor& out, const Tensor& log2_sum, const Tensor& rest, const Tensor& q_ptr,
                                           const Tensor& k_ptr, const OptTensor& k_len, bool causal, double scale) {
    refuse_tangents("oeq_amd::packed_attention_backward", grad, q, k, v, out, log2_sum, rest);
    if (records(grad, q, k, v)) {
        const auto g = PackedAttentionGradient::apply(grad, q, k, v, out, log2_sum, rest, q_ptr, k_ptr, k_len, causal, scale);
        return {g[0], g[1], g[2]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(packed_attention_backward).call(grad, q, k, v, out, log2_sum, rest, q_ptr, k_ptr, k_len, causal, scale);
}

void check_table(const Tensor& table) {
    TORCH_CHECK(!records(table), "qk_norm_rotary: the table has no gradient (pass table.detach())");
}

Tensor2 qk_norm_rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& table,
                                const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved) {
    refuse_tangents("oeq_amd::qk_norm_rotary", q, k, table, q_weight, k_weight);
    check_table(table);
    if (records(q, k, q_weight, k_weight)) {
        const auto out = QkNormRotary::apply(q, k, positions, table, q_weight, k_weight, eps, interleaved);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(qk_norm_rotary).call(q, k, positions, table, q_weight, k_weight, eps, interleaved);
}

struct QkNormRotaryGradient : public torch::autograd::Function<QkNormRotaryGradient> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q_grad, const Tensor& k_grad, const Tensor& q,
                                 const Tensor& k, const Tensor& positions, const Tensor& table, const OptTensor& q_weight,
                                 const OptTensor& k_weight, double eps, bool interleaved) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->set_materialize_grads(false);
        auto [dq, dk, dqw, dkw] = OEQ_OP(qk_norm_rotary_backward)
                                      .call(q_grad, k_grad, q, k, positions, table, q_weight, k_weight, eps, interleaved);
        return {dq, dk, dqw, dkw};
    }
    static variable_list backward(AutogradContext*, variable_list) {
        TORCH_CHECK(false, "Trying to backward through oeq_amd::qk_norm_rotary_backward but no autograd formula was registered.");
    }
};

Tensor4 qk_norm_rotary_backward_autograd(const Tensor& q_grad, const Tensor& k_grad, const Tensor& q, const Tensor& k,
                                         const Tensor& positions, const Tensor& table, const OptTensor& q_weight,
                                         const OptTensor& k_weight, double eps, bool interleaved) {
    refuse_tangents("oeq_amd::qk_norm_rotary_backward", q_grad, k_grad, q, k, table, q_weight, k_weight);
    check_table(table);
    if (records(q_grad, k_grad, q, k, q_weight, k_weight)) {
        const auto g = QkNormRotaryGradient::apply(q_grad, k_grad, q, k, positions, table, q_weight, k_weight, eps, interleaved);
        return {g[0], g[1], g[2], g[3]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(qk_norm_rotary_backward)
        .call(q_grad, k_grad, q, k, positions, table, q_weight, k_weight, eps, interleaved);
}

// Serving only: a cache that is written in place has no gradient.
Tensor qk_norm_rotary_append_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions,
                                      const Tensor& table, const Tensor& k_cache, const Tensor& v_cache, const Tensor& slots,
                                      const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved) {
    refuse_tangents("oeq_amd::qk_norm_rotary_append", q, k, v, table, k_cache, v_cache, q_weight, k_weight);
    TORCH_CHECK(!records(q, k, v, k_cache, v_cache, q_weight, k_weight),
                "qk_norm_rotary_append writes into the caches and has no gradient: call it under torch.no_grad(), or ",
                "qk_norm_rotary where gradients are needed");
    at::AutoDispatchBelowAutograd below;
    return OEQ_OP(qk_norm_rotary_append)
        .call(q, k, v, positions, table, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved);
}

// Also in inference mode, which skips the function above: a cache that autograd has saved is known to have changed.
Tensor qk_norm_rotary_append_in_place(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions,
                                      const Tensor& table, const Tensor& k_cache, const Tensor& v_cache, const Tensor& slots,
                                      const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor out = OEQ_OP(qk_norm_rotary_append)
        .call(q, k, v, positions, table, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved);
    for (const Tensor& cache : {k_cache, v_cache})
        if (!cache.is_inference()) cache.unsafeGetTensorImpl()->bump_version();
    return out;
}

Tensor irrep_dropout_autograd(const Tensor& x, const OptTensor& residual, const Tensor& channels, const Tensor& seed, double p) {
    if (has_tangent(x, residual)) {  // linear in x and the residual, and so is what a tangent becomes
        const Tensor tx = tangent_of(x), tr = tangent_of(residual);
        const OptTensor base = residual.has_value() ? OptTensor(residual->_fw_primal(0)) : OptTensor();
        const Tensor out = OEQ_OP(irrep_dropout).call(x._fw_primal(0), base, channels, seed, p);
        return at::_make_dual(out, tx.defined() ? OEQ_OP(irrep_dropout).call(tx, optional_of(tr), channels, seed, p) : tr, 0);
    }
    if (records(x, residual)) return IrrepDropout::apply(x, residual, channels, seed, p);
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(irrep_dropout).call(x, residual, channels, seed, p);
}

}  // namespace

TORCH_LIBRARY_IMPL(oeq_amd, CUDA, m) {
    m.impl("packed_attention", packed_attention_gpu);
    m.impl("packed_attention_backward", packed_attention_backward_gpu);
    m.impl("qk_norm_rotary", qk_norm_rotary_gpu);
    m.impl("qk_norm_rotary_backward", qk_norm_rotary_backward_gpu);
    m.impl("qk_norm_rotary_append", qk_norm_rotary_append_gpu);
    m.impl("irrep_dropout", irrep_dropout_gpu);
}

TORCH_LIBRARY_IMPL(oeq_amd, Autograd, m) {
    m.impl("packed_attention", packed_attention_autograd);
    m.impl("packed_attention_backward", packed_attention_backward_autograd);
    m.impl("qk_norm_rotary", qk_norm_rotary_autograd);
    m.impl("qk_norm_rotary_backward", qk_norm_rotary_backward_autograd);
    m.impl("qk_norm_rotary_append", qk_norm_rotary_append_autograd);
    m.impl("irrep_dropout", irrep_dropout_autograd);
}

TORCH_LIBRARY_IMPL(oeq_amd, ADInplaceOrView, m) { m.impl("qk_norm_rotary_append", qk_norm_rotary_append_in_place); }
