// The torch ops whose parameters are chosen row by row: checks, allocation, launches through the C ABI and autograd.
// (Schemas and fake kernels: _torch/typed.py.) Embeddings and linear layers by type are differentiable to any order: their
// gradients are ops whose own gradients are made of the same ops. Second derivatives of adapters are refused.
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

int element_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return OEQ_FLOAT32;
        case at::kHalf: return OEQ_FLOAT16;
        case at::kBFloat16: return OEQ_BFLOAT16;
        default:
            TORCH_CHECK(false, "Dtype mismatch for tensor '", name, "'. Expected: float32, float16 or bfloat16. Got: ",
                        at::toString(t.scalar_type()));
    }
}

void check_types(const Tensor& types, const Tensor& beside) {
    TORCH_CHECK(types.dim() == 1, "Shape mismatch for tensor 'types'. Expected: [rows]. Got: ", types.sizes());
    check_tensor(types, types.sizes(), at::kLong, "types", beside);
}

void check_whole(const OptTensor& order, const OptTensor& ptr) {
    TORCH_CHECK(order.has_value() == ptr.has_value(), "an index has both 'order' and 'ptr'");
}

void check_index(const Tensor& types, int64_t count, const OptTensor& order, const OptTensor& ptr) {
    check_whole(order, ptr);
    if (!order.has_value()) return;
    check_tensor(*order, {types.size(0)}, at::kInt, "order", types);
    check_tensor(*ptr, {count + 1}, at::kInt, "ptr", types);
}

// The index of a batch's types: the caller's, or one made when a call needs it.
struct Groups {
    Tensor types, order, ptr;
    int64_t count;
    Groups(const Tensor& types_, int64_t count_, const OptTensor& order_, const OptTensor& ptr_);
    void make();
    void set(oeq_typed_rows& a) {
        if (!oeq_typed_needs_index(&a)) return;
        make();
        a.order = order.data_ptr<int32_t>(), a.ptr = ptr.data_ptr<int32_t>();
    }
};

Tensor2 group_rows_gpu(const Tensor& types, int64_t count) {
    check_types(types, types);
    TORCH_CHECK(count >= 0, "group_rows: a number of types of ", count);
    OnDevice dev(types);
    const Tensor t = types.contiguous();
    const auto ints = types.options().dtype(at::kInt);
    Tensor order = at::empty({t.size(0)}, ints), ptr = at::empty({count + 1}, ints);
    const size_t nb = oeq_group_rows_workspace_bytes(t.size(0), count);
    Tensor ws;
    if (nb) ws = scratch(types, nb);
    check(oeq_group_rows(t.size(0), count, t.data_ptr<int64_t>(), order.data_ptr<int32_t>(), ptr.data_ptr<int32_t>(),
                         nb ? ws.data_ptr() : nullptr, nb, dev.stream),
          "oeq_group_rows");
    return {order, ptr};
}

Groups::Groups(const Tensor& types_, int64_t count_, const OptTensor& order_, const OptTensor& ptr_)
    : types(types_.contiguous()), count(count_) {
    check_index(types, count, order_, ptr_);
    if (order_.has_value()) order = order_->contiguous(), ptr = ptr_->contiguous();
}

void Groups::make() {
    if (!order.defined()) std::tie(order, ptr) = group_rows_gpu(types, count);
}

// Rows as the kernels take them: elements one after the other, everything else strided. (Where strides or the first
// element are not at multiples of 16 bytes the kernels go by elements.)
struct Strided {
    Tensor t;
    int64_t row = 0, part = 0, parts = 1;
    explicit Strided(const Tensor& x) : t(x) {
        const int64_t last = x.dim() - 1;
        const auto far = [&](int64_t dim) { return x.size(dim) > 1 && x.stride(dim) > INT32_MAX / 4; };  // (the C library refuses it)
        if ((x.size(last) > 1 && x.stride(last) != 1) || far(0) || far(last - 1)) t = x.contiguous();
        row = t.size(0) > 1 ? t.stride(0) : 0;
        if (last == 2) {
            parts = t.size(1);
            part = parts > 1 ? t.stride(1) : 0;
        }
    }
};

// Matrices by type, [types, outer, inner], whichever of the last two dimensions is contiguous.
struct Matrices {
    Tensor t;
    bool inner_first;  // the inner dimension is the contiguous one
    int64_t type, row;
    explicit Matrices(const Tensor& w) : t(w) {
        const int64_t d = w.dim() - 1;
        inner_first = w.size(d) <= 1 || w.stride(d) == 1;
        if (!inner_first && w.size(d - 1) > 1 && w.stride(d - 1) != 1) t = w.contiguous(), inner_first = true;
        type = d == 2 && t.size(0) > 1 ? t.stride(0) : 0;
        const int64_t other = inner_first ? d - 1 : d;
        row = t.size(other) > 1 ? t.stride(other) : 0;
    }
};

// ---------------------------------------------------------------------------
// embedding
// ---------------------------------------------------------------------------

void check_table(const Tensor& weight) {
    TORCH_CHECK(weight.dim() == 2, "Shape mismatch for tensor 'weight'. Expected: [types, channels]. Got: ", weight.sizes());
    check_tensor(weight, weight.sizes(), weight.scalar_type(), "weight", weight);
}

// (the lookup needs no index: one that is passed is checked all the same)
Tensor type_embedding_gpu(const Tensor& types, const Tensor& weight, double scale, const OptTensor& order, const OptTensor& ptr) {
    check_table(weight);
    const int type = element_of(weight, "weight");
    check_types(types, weight);
    check_index(types, weight.size(0), order, ptr);
    OnDevice dev(weight);
    const Tensor at = types.contiguous();
    const Strided table(weight);
    Tensor out = at::empty({types.size(0), weight.size(1)}, weight.options());
    check(oeq_type_lookup(type, types.size(0), weight.size(0), weight.size(1), at.data_ptr<int64_t>(), table.t.data_ptr(), table.row,
                          scale, out.data_ptr(), dev.stream),
          "oeq_type_lookup");
    return out;
}

// Sums of rows [rows, channels] or [rows, parts, channels] by type.
Tensor type_sum(const Tensor& x, Groups& index, double scale, void* stream) {
    const Strided rows(x);
    const int64_t channels = x.size(-1), count = index.count;
    index.make();
    Tensor out = at::empty({count, channels}, x.options());
    if (rows.parts == 0) return out.zero_();
    const size_t nb = oeq_type_sum_workspace_bytes(x.size(0), count, channels);
    Tensor ws;
    if (nb) ws = scratch(x, nb);
    check(oeq_type_sum(element_of(x, "grad"), x.size(0), rows.parts, count, channels, index.types.data_ptr<int64_t>(),
                       index.order.data_ptr<int32_t>(), index.ptr.data_ptr<int32_t>(), rows.t.data_ptr(), rows.row, rows.part,
                       scale, out.data_ptr(), nb ? ws.data_ptr() : nullptr, nb, stream),
          "oeq_type_sum");
    return out;
}

Tensor type_embedding_backward_gpu(const Tensor& grad, const Tensor& types, int64_t count, double scale, const OptTensor& order,
                                   const OptTensor& ptr) {
    TORCH_CHECK(grad.dim() == 2, "Shape mismatch for tensor 'grad'. Expected: [rows, channels]. Got: ", grad.sizes());
    element_of(grad, "grad");
    check_types(types, grad);
    check_tensor(grad, {types.size(0), grad.size(1)}, grad.scalar_type(), "grad", grad);
    OnDevice dev(grad);
    Groups index(types, count, order, ptr);
    return type_sum(grad, index, scale, dev.stream);
}

// ---------------------------------------------------------------------------
// linear layers by type
// ---------------------------------------------------------------------------

void check_linear(const Tensor& x, const Tensor& weight, const Tensor& types) {
    TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "Shape mismatch for tensor 'x'. Expected: [rows, channels] or [rows, components, ",
                "channels]. Got: ", x.sizes());
    element_of(x, "x");
    TORCH_CHECK(weight.dim() == 3 && weight.size(2) == x.size(-1), "Shape mismatch for tensor 'weight'. Expected: [types, out, ",
                x.size(-1), "]. Got: ", weight.sizes());
    check_tensor(x, x.sizes(), x.scalar_type(), "x", x);
    check_tensor(weight, weight.sizes(), x.scalar_type(), "weight", x);
    TORCH_CHECK(types.dim() == 1, "Shape mismatch for tensor 'types'. Expected: [rows]. Got: ", types.sizes());
    check_tensor(types, {x.size(0)}, at::kLong, "types", x);
}

// (the index is set where a product needs one)
oeq_typed_rows rows_of(const Tensor& like, const Strided& x, const Tensor& type_of_row, int64_t types, int64_t inner, int64_t outer) {
    oeq_typed_rows a{};
    a.type = element_of(like, "x");
    a.rows = like.size(0), a.parts = x.parts, a.types = types, a.inner = inner, a.outer = outer;
    a.x_row_stride = x.row, a.x_part_stride = x.part, a.x = x.t.data_ptr();
    a.type_of_row = type_of_row.data_ptr<int64_t>();
    return a;
}

void set_matrices(oeq_typed_rows& a, const Matrices& w, bool across) {
    a.w = w.t.data_ptr(), a.w_type_stride = w.type, a.w_row_stride = w.row, a.across = across;
}

// sum over rows of a^T b by type, of elements like `like`.
Tensor typed_sum(const Tensor& a_, const Tensor& b_, int thin, int64_t a_columns, int64_t b_columns, const Tensor& like,
                 Groups& index, void* stream) {
    const Strided a(a_), b(b_);
    const int64_t types = index.count;
    index.make();
    Tensor out = at::empty({types, a_columns, b_columns}, like.options());
    if (a.parts == 0) return out.zero_();
    oeq_typed_sum d{};
    d.type = element_of(like, "x"), d.thin = thin;
    d.rows = a_.size(0), d.parts = a.parts, d.types = types, d.a_columns = a_columns, d.b_columns = b_columns;
    d.a_row_stride = a.row, d.a_part_stride = a.part, d.b_row_stride = b.row, d.b_part_stride = b.part;
    d.a = a.t.data_ptr(), d.b = b.t.data_ptr();
    d.order = index.order.data_ptr<int32_t>(), d.ptr = index.ptr.data_ptr<int32_t>();
    const size_t nb = oeq_typed_sum_workspace_bytes(&d);
    Tensor ws;
    if (nb) ws = scratch(like, nb);
    check(oeq_typed_sum_products(&d, out.data_ptr(), nb ? ws.data_ptr() : nullptr, nb, stream), "oeq_typed_sum_products");
    return out;
}

std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = last;
    return shape;
}

Tensor typed_linear_gpu(const Tensor& x, const Tensor& weight, const Tensor& types, const OptTensor& bias, const OptTensor& order,
                        const OptTensor& ptr) {
    check_linear(x, weight, types);
    if (bias.has_value()) check_tensor(*bias, {weight.size(0), weight.size(1)}, x.scalar_type(), "bias", x);
    OnDevice dev(x);
    Tensor out = at::empty(with_last(x, weight.size(1)), x.options());
    if (out.numel() == 0) return out;
    Groups index(types, weight.size(0), order, ptr);
    const Strided in(x);
    const Matrices w(weight);
    Tensor b;
    if (bias.has_value()) b = bias->contiguous();
    oeq_typed_rows a = rows_of(x, in, index.types, weight.size(0), weight.size(2), weight.size(1));
    set_matrices(a, w, !w.inner_first);
    index.set(a);
    a.bias = b.defined() ? b.data_ptr() : nullptr;
    check(oeq_typed_product(&a, out.data_ptr(), dev.stream), "oeq_typed_product");
    return out;
}

// (gradients that are not wanted are empty tensors)
Tensor3 typed_linear_backward_gpu(const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& types,
                                  const OptTensor& order, const OptTensor& ptr, bool want_x, bool want_weight, bool want_bias) {
    check_linear(x, weight, types);
    check_tensor(grad, with_last(x, weight.size(1)), x.scalar_type(), "grad", x);
    OnDevice dev(x);
    const int64_t count = weight.size(0), outer = weight.size(1), inner = weight.size(2);
    Groups index(types, count, order, ptr);
    const auto none = [&] { return at::empty({0}, x.options()); };
    Tensor dx = want_x ? at::empty(x.sizes(), x.options()) : none(), dw, db;
    if (want_x) {
        if (dx.numel()) {
            const Strided g(grad);
            const Matrices w(weight);
            oeq_typed_rows a = rows_of(x, g, index.types, count, outer, inner);
            set_matrices(a, w, w.inner_first);
            index.set(a);
            check(oeq_typed_product(&a, dx.data_ptr(), dev.stream), "oeq_typed_product");
        }
    }
    dw = want_weight ? typed_sum(grad, x, 0, outer, inner, x, index, dev.stream) : none();
    db = want_bias ? type_sum(grad, index, 1.0, dev.stream) : none();
    return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// low-rank adapters
// ---------------------------------------------------------------------------

void check_adapters(const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up, const Tensor& types,
                    const OptTensor& scale) {
    TORCH_CHECK(x.dim() == 2, "Shape mismatch for tensor 'x'. Expected: [rows, channels]. Got: ", x.sizes());
    element_of(x, "x");
    check_tensor(x, x.sizes(), x.scalar_type(), "x", x);
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x.size(1), "Shape mismatch for tensor 'weight'. Expected: [out, ", x.size(1),
                "]. Got: ", weight.sizes());
    check_tensor(weight, weight.sizes(), x.scalar_type(), "weight", x);
    TORCH_CHECK(down.dim() == 3 && down.size(2) == x.size(1), "Shape mismatch for tensor 'down'. Expected: [adapters, rank, ", x.size(1),
                "]. Got: ", down.sizes());
    check_tensor(down, down.sizes(), x.scalar_type(), "down", x);
    check_tensor(up, {down.size(0), weight.size(0), down.size(1)}, x.scalar_type(), "up", x);
    check_tensor(types, {x.size(0)}, at::kLong, "adapters", x);
    if (scale.has_value()) check_tensor(*scale, {down.size(0)}, at::kFloat, "scale", x);
}

// The thin product beside shared weights: matrices [types, .., ..] with the given dimensions of outer channels and rank.
void set_thin(oeq_typed_rows& a, const Tensor& thin, const Tensor& matrices, int outer, int rank) {
    a.shared = 1, a.rank = (int32_t)matrices.size(rank), a.thin = thin.data_ptr<float>(), a.up = matrices.data_ptr();
    a.up_type_stride = matrices.stride(0), a.up_outer_stride = matrices.stride(outer), a.up_rank_stride = matrices.stride(rank);
}

// thin = scale_t m_t x, [rows, stride] in float.
Tensor thin_product(const Tensor& x, const Tensor& matrices, bool transposed, const OptTensor& scale, Groups& index,
                    void* stream) {
    const Matrices w(matrices);
    const Strided in(x);
    const int64_t rank = matrices.size(transposed ? 2 : 1), inner = matrices.size(transposed ? 1 : 2);
    Tensor out = at::empty({x.size(0), oeq_thin_stride(rank)}, x.options().dtype(at::kFloat));
    if (out.numel() == 0) return out;
    oeq_typed_rows a = rows_of(x, in, index.types, matrices.size(0), inner, rank);
    set_matrices(a, w, w.inner_first == transposed);
    index.set(a);
    const Tensor by = scale.has_value() ? scale->contiguous() : Tensor();
    check(oeq_typed_thin_product(&a, by.defined() ? by.data_ptr<float>() : nullptr, out.data_ptr<float>(), stream), "oeq_typed_thin_product");
    return out;
}

// (out, thin): the second is kept for the backward pass.
Tensor2 adapter_linear_gpu(const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up, const Tensor& types,
                           const OptTensor& scale, const OptTensor& order, const OptTensor& ptr) {
    check_adapters(x, weight, down, up, types, scale);
    OnDevice dev(x);
    const int64_t count = down.size(0), rank = down.size(1);
    Groups index(types, count, order, ptr);
    Tensor thin = thin_product(x, down, false, scale, index, dev.stream);
    Tensor out = at::empty({x.size(0), weight.size(0)}, x.options());
    if (out.numel() == 0) return {out, thin};
    const Strided in(x);
    const Matrices w(weight);
    oeq_typed_rows a = rows_of(x, in, index.types, count, weight.size(1), weight.size(0));
    set_matrices(a, w, !w.inner_first);
    set_thin(a, thin, up, 1, 2);
    index.set(a);
    check(oeq_typed_product(&a, out.data_ptr(), dev.stream), "oeq_typed_product");
    return {out, thin};
}

Tensor4 adapter_linear_backward_gpu(const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up,
                                    const Tensor& types, const OptTensor& scale, const Tensor& thin, const OptTensor& order,
                                    const OptTensor& ptr, bool want_x, bool want_weight, bool want_down, bool want_up) {
    check_adapters(x, weight, down, up, types, scale);
    const int64_t count = down.size(0), rank = down.size(1), inner = weight.size(1), outer = weight.size(0);
    check_tensor(grad, {x.size(0), outer}, x.scalar_type(), "grad", x);
    check_tensor(thin, {x.size(0), oeq_thin_stride(rank)}, at::kFloat, "thin", x);
    OnDevice dev(x);
    Groups index(types, count, order, ptr);
    const Tensor u = thin.contiguous();
    const auto none = [&] { return at::empty({0}, x.options()); };
    Tensor dx = want_x ? at::empty(x.sizes(), x.options()) : none(), dw, ddown, dup, v;
    if (want_x || want_down) v = thin_product(grad, up, true, scale, index, dev.stream);
    if (want_x) {
        if (dx.numel()) {
            const Strided g(grad);
            const Matrices w(weight);
            oeq_typed_rows a = rows_of(x, g, index.types, count, outer, inner);
            set_matrices(a, w, w.inner_first);
            set_thin(a, v, down, 2, 1);
            index.set(a);
            check(oeq_typed_product(&a, dx.data_ptr(), dev.stream), "oeq_typed_product");
        }
    }
    ddown = want_down ? typed_sum(v, x, 1, rank, inner, x, index, dev.stream) : none();
    dup = want_up ? typed_sum(grad, u, 2, outer, rank, x, index, dev.stream) : none();
    if (want_weight) {
        const Tensor one = at::zeros({x.size(0)}, types.options());  // (all rows are of one type)
        Groups all(one, 1, {}, {});
        dw = typed_sum(grad, x, 0, outer, inner, x, all, dev.stream).squeeze(0);
    } else {
        dw = none();
    }
    return {dx, dw, ddown, dup};
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

Tensor tensor_of(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// The index of a call that will be differentiated: made now, so that the backward pass finds it.
Tensor2 recorded_index(const Tensor& types, int64_t count, const OptTensor& order, const OptTensor& ptr) {
    check_whole(order, ptr);
    if (order.has_value()) return {*order, *ptr};
    return OEQ_OP(group_rows).call(types, count);
}

struct TypeEmbedding : public torch::autograd::Function<TypeEmbedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& types, double scale, const OptTensor& order_,
                          const OptTensor& ptr_) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [order, ptr] = recorded_index(types, weight.size(0), order_, ptr_);
        ctx->save_for_backward({types, order, ptr});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["count"] = weight.size(0);
        ctx->set_materialize_grads(false);
        return OEQ_OP(type_embedding).call(types, weight, scale, order, ptr);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        out[0] = OEQ_OP(type_embedding_backward)
                     .call(grads[0], s[0], ctx->saved_data["count"].toInt(), ctx->saved_data["scale"].toDouble(), s[1], s[2]);
        return out;
    }
};

Tensor type_embedding_autograd(const Tensor& types, const Tensor& weight, double scale, const OptTensor& order, const OptTensor& ptr) {
    refuse_tangents("oeq_amd::type_embedding", weight);
    if (records(weight)) return TypeEmbedding::apply(weight, types, scale, order, ptr);
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(type_embedding).call(types, weight, scale, order, ptr);
}

// The sum of rows by type is linear: its gradient is the lookup.
struct TypeEmbeddingGradient : public torch::autograd::Function<TypeEmbeddingGradient> {
    static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& types, int64_t count, double scale,
                          const OptTensor& order_, const OptTensor& ptr_) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [order, ptr] = recorded_index(types, count, order_, ptr_);
        ctx->save_for_backward({types, order, ptr});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return OEQ_OP(type_embedding_backward).call(grad, types, count, scale, order, ptr);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        out[0] = OEQ_OP(type_embedding).call(s[0], grads[0], ctx->saved_data["scale"].toDouble(), s[1], s[2]);
        return out;
    }
};

Tensor type_embedding_backward_autograd(const Tensor& grad, const Tensor& types, int64_t count, double scale, const OptTensor& order,
                                        const OptTensor& ptr) {
    refuse_tangents("oeq_amd::type_embedding_backward", grad);
    if (records(grad)) return TypeEmbeddingGradient::apply(grad, types, count, scale, order, ptr);
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(type_embedding_backward).call(grad, types, count, scale, order, ptr);
}

struct TypedLinear : public torch::autograd::Function<TypedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& types, const OptTensor& bias,
                          const OptTensor& order_, const OptTensor& ptr_) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [order, ptr] = recorded_index(types, weight.size(0), order_, ptr_);
        ctx->save_for_backward({x, weight, types, order, ptr});
        ctx->saved_data["bias"] = bias.has_value();
        ctx->set_materialize_grads(false);
        return OEQ_OP(typed_linear).call(x, weight, types, bias, order, ptr);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        const bool bias = ctx->saved_data["bias"].toBool();
        // (edges are counted over the tensors that were there: x, weight, types, bias)
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = bias && ctx->needs_input_grad(3);
        auto [dx, dw, db] =
            OEQ_OP(typed_linear_backward).call(grads[0], s[0], s[1], s[2], s[3], s[4], want_x, want_w, want_b);
        if (want_x) out[0] = dx;
        if (want_w) out[1] = dw;
        if (want_b) out[3] = db;
        return out;
    }
};

Tensor typed_linear_autograd(const Tensor& x, const Tensor& weight, const Tensor& types, const OptTensor& bias, const OptTensor& order,
                             const OptTensor& ptr) {
    refuse_tangents("oeq_amd::typed_linear", x, weight, bias);
    if (records(x, weight, bias)) return TypedLinear::apply(x, weight, types, bias, order, ptr);
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(typed_linear).call(x, weight, types, bias, order, ptr);
}

// dx_i = g_i W_t, dW_t = sum g_i^T x_i, db_t = sum g_i are linear in each of g, x and W: with cotangents a, b, c of them
// g gets a_i W_t^T + x_i b_t^T + c_t, x gets g_i b_t and W gets sum g_i^T a_i.
struct TypedLinearGradient : public torch::autograd::Function<TypedLinearGradient> {
    static variable_list forward(AutogradContext* ctx, const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& types,
                                 const OptTensor& order_, const OptTensor& ptr_, bool want_x, bool want_weight, bool want_bias) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [order, ptr] = recorded_index(types, weight.size(0), order_, ptr_);
        ctx->save_for_backward({grad, x, weight, types, order, ptr});
        ctx->saved_data["want_x"] = want_x;
        ctx->saved_data["want_weight"] = want_weight;
        ctx->saved_data["want_bias"] = want_bias;
        ctx->set_materialize_grads(false);
        auto [dx, dw, db] = OEQ_OP(typed_linear_backward).call(grad, x, weight, types, order, ptr, want_x, want_weight, want_bias);
        return {dx, dw, db};
    }
    static variable_list backward(AutogradContext* ctx, variable_list cotangents) {
        variable_list out(9);
        const auto s = ctx->get_saved_variables();
        const Tensor &grad = s[0], &x = s[1], &weight = s[2], &types = s[3];
        const OptTensor order = s[4], ptr = s[5];
        const Tensor a = ctx->saved_data["want_x"].toBool() ? cotangents[0] : Tensor();
        const Tensor b = ctx->saved_data["want_weight"].toBool() ? cotangents[1] : Tensor();
        const Tensor c = ctx->saved_data["want_bias"].toBool() ? cotangents[2] : Tensor();
        if (ctx->needs_input_grad(0)) {
            Tensor g;
            if (a.defined()) g = OEQ_OP(typed_linear).call(a, weight, types, {}, order, ptr);
            if (b.defined() || c.defined()) {
                Tensor more;
                if (b.defined()) {
                    more = OEQ_OP(typed_linear).call(x, b, types, optional_of(c), order, ptr);
                } else {  // (no product with zeros: what a row holds has no part in c_t)
                    more = OEQ_OP(type_embedding).call(types, c, 1.0, order, ptr);
                    if (grad.dim() == 3) more = more.unsqueeze(1).expand_as(grad);
                }
                g = g.defined() ? g + more : more;
            }
            out[0] = g;
        }
        if (ctx->needs_input_grad(1) && b.defined())
            out[1] = std::get<0>(OEQ_OP(typed_linear_backward).call(grad, x, b, types, order, ptr, true, false, false));
        if (ctx->needs_input_grad(2) && a.defined())
            out[2] = std::get<1>(OEQ_OP(typed_linear_backward).call(grad, a, weight, types, order, ptr, false, true, false));
        return out;
    }
};

Tensor3 typed_linear_backward_autograd(const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& types,
                                       const OptTensor& order, const OptTensor& ptr, bool want_x, bool want_weight, bool want_bias) {
    refuse_tangents("oeq_amd::typed_linear_backward", grad, x, weight);
    if (records(grad, x, weight)) {
        const auto g = TypedLinearGradient::apply(grad, x, weight, types, order, ptr, want_x, want_weight, want_bias);
        return {g[0], g[1], g[2]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(typed_linear_backward).call(grad, x, weight, types, order, ptr, want_x, want_weight, want_bias);
}

struct AdapterLinear : public torch::autograd::Function<AdapterLinear> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up,
                                 const Tensor& types, const OptTensor& scale, const OptTensor& order_, const OptTensor& ptr_) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [order, ptr] = recorded_index(types, down.size(0), order_, ptr_);
        auto [out, thin] = OEQ_OP(adapter_linear).call(x, weight, down, up, types, scale, order, ptr);
        ctx->save_for_backward({x, weight, down, up, types, tensor_of(scale), thin, order, ptr});
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({thin});
        return {out, thin};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(8);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        bool want[4];
        for (int i = 0; i < 4; ++i) want[i] = ctx->needs_input_grad(i);
        auto [dx, dw, ddown, dup] = OEQ_OP(adapter_linear_backward)
                                        .call(grads[0], s[0], s[1], s[2], s[3], s[4], optional_of(s[5]), s[6], s[7], s[8], want[0], want[1], want[2], want[3]);
        if (want[0]) out[0] = dx;
        if (want[1]) out[1] = dw;
        if (want[2]) out[2] = ddown;
        if (want[3]) out[3] = dup;
        return out;
    }
};

Tensor2 adapter_linear_autograd(const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up, const Tensor& types,
                                const OptTensor& scale, const OptTensor& order, const OptTensor& ptr) {
    refuse_tangents("oeq_amd::adapter_linear", x, weight, down, up, scale);
    TORCH_CHECK(!records(scale), "adapter_linear: the scales have no gradient (pass scale.detach())");
    if (records(x, weight, down, up)) {
        const auto out = AdapterLinear::apply(x, weight, down, up, types, scale, order, ptr);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(adapter_linear).call(x, weight, down, up, types, scale, order, ptr);
}

struct AdapterLinearGradient : public torch::autograd::Function<AdapterLinearGradient> {
    static variable_list forward(AutogradContext* ctx, const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& down,
                                 const Tensor& up, const Tensor& types, const OptTensor& scale, const Tensor& thin, const OptTensor& order,
                                 const OptTensor& ptr, bool want_x, bool want_weight, bool want_down, bool want_up) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->set_materialize_grads(false);
        auto [dx, dw, ddown, dup] = OEQ_OP(adapter_linear_backward)
                                        .call(grad, x, weight, down, up, types, scale, thin, order, ptr, want_x, want_weight, want_down, want_up);
        return {dx, dw, ddown, dup};
    }
    static variable_list backward(AutogradContext*, variable_list) {
        TORCH_CHECK(false, "Trying to backward through oeq_amd::adapter_linear_backward but no autograd formula was registered.");
    }
};

Tensor4 adapter_linear_backward_autograd(const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up,
                                         const Tensor& types, const OptTensor& scale, const Tensor& thin, const OptTensor& order,
                                         const OptTensor& ptr, bool want_x, bool want_weight, bool want_down, bool want_up) {
    refuse_tangents("oeq_amd::adapter_linear_backward", grad, x, weight, down, up, scale, thin);
    if (records(grad, x, weight, down, up)) {
        const auto g = AdapterLinearGradient::apply(grad, x, weight, down, up, types, scale, thin, order, ptr, want_x, want_weight,
                                                    want_down, want_up);
        return {g[0], g[1], g[2], g[3]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return OEQ_OP(adapter_linear_backward)
        .call(grad, x, weight, down, up, types, scale, thin, order, ptr, want_x, want_weight, want_down, want_up);
}

}  // namespace

TORCH_LIBRARY_IMPL(oeq_amd, CUDA, m) {
    m.impl("group_rows", group_rows_gpu);
    m.impl("type_embedding", type_embedding_gpu);
    m.impl("type_embedding_backward", type_embedding_backward_gpu);
    m.impl("typed_linear", typed_linear_gpu);
    m.impl("typed_linear_backward", typed_linear_backward_gpu);
    m.impl("adapter_linear", adapter_linear_gpu);
    m.impl("adapter_linear_backward", adapter_linear_backward_gpu);
}

TORCH_LIBRARY_IMPL(oeq_amd, Autograd, m) {
    m.impl("type_embedding", type_embedding_autograd);
    m.impl("type_embedding_backward", type_embedding_backward_autograd);
    m.impl("typed_linear", typed_linear_autograd);
    m.impl("typed_linear_backward", typed_linear_backward_autograd);
    m.impl("adapter_linear", adapter_linear_autograd);
    m.impl("adapter_linear_backward", adapter_linear_backward_autograd);
}
