// PyTorch module `sc_dense`: the dense 8-bit layers and the distillation loss of libgeo_sc.so on tensors.  Checks, outputs
// and workspaces from the caching allocator, launch on PyTorch's current HIP stream.  In C++ because a single
// token's call is bound by its host time.
#include "sc_torch_common.h"

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>

using namespace geo_sc_torch;

namespace {

using MaybeTensor = std::optional<at::Tensor>;

int dtype_of(at::ScalarType t, const char* what)
{
    switch (t) {
    case at::kFloat: return GEO_SC_F32;
    case at::kBFloat16: return GEO_SC_BF16;
    case at::kHalf: return GEO_SC_F16;
    default: TORCH_CHECK(false, what, " must be float32, bfloat16 or float16, got ", t);
    }
}

void on_gpu(const at::Tensor& t, const char* what)
{
    TORCH_CHECK(t.is_cuda(), what, " must be on the GPU");
    TORCH_CHECK(t.layout() == at::kStrided && !t.is_neg(), what, " must be an ordinary dense tensor");
    TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), what, " carries a forward-mode tangent, which these operators have no rule for");
}
void with(const at::Tensor& t, const char* what, const at::Tensor& other, const char* other_what)
{
    on_gpu(t, what);
    TORCH_CHECK(t.device() == other.device(), what, " and ", other_what, " are on different devices");
}

// Whoever records a program's operations to run them again sees the allocation of the outputs, and not what fills them.
void not_recorded()
{
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                "the dense 8-bit layers and the distillation loss cannot be traced");
}

geo_sc_stream_t stream_of(const at::Tensor& t)
{
    return (geo_sc_stream_t)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// A tensor of any number of dimensions as rows of its last one, with a distance between them; copied only where its strides
// have no such form.
struct Rows {
    at::Tensor t;
    int64_t rows, cols, stride;
};
Rows as_rows(const at::Tensor& t, const char* what)
{
    on_gpu(t, what);
    TORCH_CHECK(t.dim() >= 1, what, " must have a dimension");
    const int64_t cols = t.size(-1);
    TORCH_CHECK(cols >= 1, what, " has rows of no elements");
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= 0) return {t, t.size(0), cols, t.size(0) > 1 ? t.stride(0) : cols};
    const at::Tensor c = t.contiguous();
    return {c, c.numel() / cols, cols, cols};
}

// A gradient that a kernel wrote.  Under create_graph it needs a graph of its own, or a second derivative would come out as zero: here
// a node that raises, on the way to all that the gradient depends on (what the node being evaluated leads to, and `upstream`).
struct Once : torch::autograd::Node {
    torch::autograd::variable_list apply(torch::autograd::variable_list&&) override
    {
        TORCH_CHECK(false, "the dense 8-bit layers and the distillation loss can be differentiated once only");
    }
    std::string name() const override { return "DifferentiableOnce"; }
};
at::Tensor once(const at::Tensor& g, std::initializer_list<at::Tensor> upstream)
{
    if (!at::GradMode::is_enabled()) return g;
    const auto current = torch::autograd::get_current_node();
    torch::autograd::edge_list edges;
    if (current) edges = current->next_edges();
    for (const at::Tensor& u : upstream)
        if (u.defined() && u.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(u));
    const auto node = std::make_shared<Once>();
    node->set_next_edges(std::move(edges));
    torch::autograd::set_history(g, node);
    return g;
}

// 8-bit rows that start at multiples of 16 bytes: what the product's fast way takes
at::Tensor empty_q(at::IntArrayRef sizes, const at::TensorOptions& options)
{
    const int64_t cols = sizes.back(), stride = (cols + 15) / 16 * 16;
    if (stride == cols) return at::empty(sizes, options.dtype(at::kChar));
    std::vector<int64_t> wide(sizes.begin(), sizes.end());
    wide.back() = stride;
    return at::empty(wide, options.dtype(at::kChar)).narrow(-1, 0, cols);
}

at::Tensor row_scalars(const at::Tensor& x) { return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)); }

void* data_of(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }

std::tuple<at::Tensor, at::Tensor, MaybeTensor> quantize_rows(const at::Tensor& x, std::optional<at::ScalarType> values_type)
{
    not_recorded();
    const Rows r = as_rows(x, "x");
    const int dtype = dtype_of(x.scalar_type(), "x"), vtype = values_type ? dtype_of(*values_type, "values") : 0;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const at::Tensor q = empty_q(x.sizes(), x.options()), scale = row_scalars(x);
    MaybeTensor values;
    if (values_type) values = at::empty(x.sizes(), x.options().dtype(*values_type));
    check_status(geo_sc_quantize_rows(r.t.const_data_ptr(), dtype, r.rows, r.cols, r.stride, q.data_ptr<int8_t>(), (r.cols + 15) / 16 * 16,
                                      scale.data_ptr<float>(), data_of(values), vtype, stream_of(x)),
                 "quantize_rows");
    return {q, scale, values};
}

// (q, scale, total, values, rstd); total is x where there is no residual
std::tuple<at::Tensor, at::Tensor, at::Tensor, MaybeTensor, MaybeTensor> rms_norm_q8(const at::Tensor& x, const at::Tensor& weight,
                                                                                   const MaybeTensor& residual, double eps,
                                                                                   std::optional<at::ScalarType> values_type,
                                                                                   bool for_backward)
{
    not_recorded();
    const Rows r = as_rows(x, "x");
    const int dtype = dtype_of(x.scalar_type(), "x"), vtype = values_type ? dtype_of(*values_type, "values") : 0;
    with(weight, "weight", x, "x");
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == r.cols, "weight must have the ", r.cols, " elements of a row of x");
    TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "weight must have the type of x");
    TORCH_CHECK(eps >= 0, "eps must not be negative");
    Rows s = {};
    if (residual) {
        with(*residual, "residual", x, "x");
        TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "residual must have the shape and type of x");
        s = as_rows(*residual, "residual");
    }
    const at::Tensor w = weight.contiguous();
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const at::Tensor q = empty_q(x.sizes(), x.options()), scale = row_scalars(x);
    const at::Tensor total = residual ? at::empty(x.sizes(), x.options()) : x;
    MaybeTensor values, rstd;
    if (values_type) values = at::empty(x.sizes(), x.options().dtype(*values_type));
    if (for_backward) rstd = at::empty({r.rows}, scale.options());
    check_status(geo_sc_rms_norm_q8(r.t.const_data_ptr(), residual ? s.t.const_data_ptr() : nullptr, w.const_data_ptr(), dtype, r.rows, r.cols,
                                    r.stride, residual ? s.stride : 0, (float)eps, q.data_ptr<int8_t>(), (r.cols + 15) / 16 * 16,
                                    scale.data_ptr<float>(), residual ? total.data_ptr() : nullptr, data_of(values), vtype,
                                    (float*)data_of(rstd), stream_of(x)),
                 "rms_norm_q8");
    return {q, scale, total, values, rstd};
}

// (dx, dweight)
std::tuple<at::Tensor, MaybeTensor> rms_norm_q8_backward(const MaybeTensor& grad_values, const MaybeTensor& grad_total,
                                                         const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight,
                                                         const at::Tensor& rstd, bool need_weight)
{
    not_recorded();
    const Rows t = as_rows(x, "x");
    Rows r = {};
    if (residual.defined()) r = as_rows(residual, "residual");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    if (!grad_values || t.rows == 0) {   // nothing comes through the norm itself
        return {grad_total ? grad_total->to(x.scalar_type()) : at::zeros_like(x),
                need_weight ? MaybeTensor(at::zeros_like(weight)) : MaybeTensor()};
    }
    const Rows g = as_rows(*grad_values, "gradient");
    Rows h = {};
    if (grad_total) h = as_rows(grad_total->to(x.scalar_type()), "gradient");
    const at::Tensor w = weight.contiguous(), dx = at::empty(x.sizes(), x.options());
    MaybeTensor dw, workspace;
    size_t bytes = 0;
    if (need_weight) {
        dw = at::empty_like(w);
        check_status(geo_sc_rms_norm_q8_backward_workspace_size(t.rows, t.cols, &bytes), "workspace query");
        workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    }
    const int dtype = dtype_of(x.scalar_type(), "x");
    check_status(geo_sc_rms_norm_q8_backward(g.t.const_data_ptr(), dtype_of(g.t.scalar_type(), "gradient"), g.stride,
                                             grad_total ? h.t.const_data_ptr() : nullptr, h.stride, t.t.const_data_ptr(), t.stride,
                                             residual.defined() ? r.t.const_data_ptr() : nullptr, r.stride, w.const_data_ptr(), dtype, t.rows,
                                             t.cols, rstd.const_data_ptr<float>(), dx.data_ptr(), data_of(dw), data_of(workspace), bytes,
                                             stream_of(x)),
                 "rms_norm_q8 backward");
    const at::Tensor sum_grad = grad_total ? *grad_total : at::Tensor();
    if (dw) once(*dw, {*grad_values});
    return {once(dx, {*grad_values, sum_grad}), dw};
}

// What the backward forms x + residual from: themselves, because `total` is rounded to their type; where that is fp32, `total`
// is the sum itself and half the reading.
std::pair<at::Tensor, at::Tensor> summands(const at::Tensor& x, const MaybeTensor& residual, const at::Tensor& total)
{
    if (residual && x.scalar_type() != at::kFloat) return {x, *residual};
    return {total, at::Tensor()};
}

// 8-bit rows with a scale each: what the products take
struct Q8 {
    Rows r;
    at::Tensor scale;
};
Q8 as_q8(const at::Tensor& q, const at::Tensor& scale, const char* what)
{
    on_gpu(q, what);
    TORCH_CHECK(q.scalar_type() == at::kChar, what, " must be int8, got ", q.scalar_type());
    Q8 v;
    if (q.dim() > 2 && q.stride(-1) == 1 && q.stride(-2) >= q.size(-1)) {
        // rows of one distance through all leading dimensions (what quantize_rows returns for odd lengths)
        bool one = true;
        for (int64_t d = q.dim() - 3; d >= 0; --d) one = one && q.stride(d) == q.stride(d + 1) * q.size(d + 1);
        if (one && q.size(-1) >= 1) v.r = {q, q.numel() / q.size(-1), q.size(-1), q.stride(-2)};
        else v.r = as_rows(q, what);
    } else {
        v.r = as_rows(q, what);
    }
    with(scale, "scale", q, what);
    TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.numel() == v.r.rows, what, ": the scales must be float32, one per row");
    v.scale = scale.contiguous();
    return v;
}

at::Tensor matmul_q8(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& wq, const at::Tensor& wscale, at::ScalarType type)
{
    not_recorded();
    const Q8 x = as_q8(q, scale, "q"), w = as_q8(wq, wscale, "weight_q");
    const int dtype = dtype_of(type, "dtype");
    with(wq, "weight_q", q, "q");
    TORCH_CHECK(wq.dim() == 2, "weight_q must be (cols, inner)");
    TORCH_CHECK(x.r.cols == w.r.cols, "rows of q have ", x.r.cols, " elements, rows of weight_q ", w.r.cols);
    TORCH_CHECK(x.r.cols <= 131071, "at most 131071 elements per row");
    std::vector<int64_t> sizes(q.sizes().begin(), q.sizes().end());
    sizes.back() = w.r.rows;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    const at::Tensor y = at::empty(sizes, q.options().dtype(type));
    if (y.numel() == 0) return y;
    size_t bytes = 0;
    check_status(geo_sc_matmul_q8_workspace_size(x.r.t.const_data_ptr<int8_t>(), x.r.stride, w.r.t.const_data_ptr<int8_t>(),
                                                 w.r.stride, x.r.rows, w.r.rows, x.r.cols, &bytes), "workspace query");
    MaybeTensor workspace;
    if (bytes) workspace = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check_status(geo_sc_matmul_q8(x.r.t.const_data_ptr<int8_t>(), x.r.stride, x.scale.const_data_ptr<float>(), w.r.t.const_data_ptr<int8_t>(),
                                  w.r.stride, w.scale.const_data_ptr<float>(), x.r.rows, w.r.rows, x.r.cols, y.data_ptr(), dtype,
                                  data_of(workspace), bytes, stream_of(q)),
                 "matmul_q8");
    return y;
}

std::tuple<MaybeTensor, MaybeTensor> matmul_q8_backward(const at::Tensor& grad, const at::Tensor& q, const at::Tensor& scale,
                                                        const at::Tensor& wq, const at::Tensor& wscale,
                                                        std::optional<at::ScalarType> dx_type, std::optional<at::ScalarType> dw_type)
{
    not_recorded();
    const Q8 x = as_q8(q, scale, "q"), w = as_q8(wq, wscale, "weight_q");
    if (w.r.rows == 0 && grad.numel() == 0) {   // no columns: sums of nothing
        on_gpu(grad, "gradient");
        return {dx_type ? MaybeTensor(at::zeros(q.sizes(), q.options().dtype(*dx_type))) : MaybeTensor(),
                dw_type ? MaybeTensor(at::empty(wq.sizes(), q.options().dtype(*dw_type))) : MaybeTensor()};
    }
    Rows g = as_rows(grad, "gradient");
    if (g.rows > 1 && g.stride && g.stride < g.cols) g = as_rows(grad.contiguous(), "gradient");   // (rows that overlap)
    with(grad, "gradient", q, "q");
    TORCH_CHECK(x.r.cols == w.r.cols && g.rows == x.r.rows && g.cols == w.r.rows, "gradient must have the shape of the product");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    MaybeTensor dx, dw;
    if (dx_type) dx = at::empty(q.sizes(), q.options().dtype(*dx_type));
    if (dw_type) dw = at::empty(wq.sizes(), q.options().dtype(*dw_type));
    if (g.rows == 0 && dw) dw->zero_();
    if (g.rows == 0 || (!dx && !dw)) return {dx, dw};
    const int grad_type = dtype_of(g.t.scalar_type(), "gradient");
    size_t bytes = 0;
    check_status(geo_sc_matmul_q8_backward_workspace_size(g.rows, g.cols, x.r.cols, grad_type, dx.has_value(), dw.has_value(), &bytes),
                 "workspace query");
    const at::Tensor workspace = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check_status(geo_sc_matmul_q8_backward(g.t.const_data_ptr(), grad_type, g.stride, x.r.t.const_data_ptr<int8_t>(), x.r.stride,
                                           x.scale.const_data_ptr<float>(), w.r.t.const_data_ptr<int8_t>(), w.r.stride,
                                           w.scale.const_data_ptr<float>(), g.rows, g.cols, x.r.cols, data_of(dx),
                                           dx ? dtype_of(*dx_type, "dx") : 0, data_of(dw), dw ? dtype_of(*dw_type, "dw") : 0,
                                           workspace.data_ptr(), bytes, stream_of(q)),
                 "matmul_q8 backward");
    if (dx) once(*dx, {grad});
    if (dw) once(*dw, {grad});
    return {dx, dw};
}

// the teacher's entries of the rows of `logits`
struct Top {
    at::Tensor logits, index;
    int top, dtype, index_bytes;
};
Top as_top(const Rows& z, const at::Tensor& logits, const at::Tensor& top_logits, const at::Tensor& top_index)
{
    with(top_logits, "top_logits", logits, "logits");
    with(top_index, "top_index", logits, "logits");
    TORCH_CHECK(top_logits.sizes() == top_index.sizes(), "top_logits and top_index must have one shape");
    TORCH_CHECK(top_logits.dim() == logits.dim() &&
                    top_logits.sizes().slice(0, logits.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                "top_logits must have the rows of logits");
    TORCH_CHECK(top_logits.size(-1) >= 1 && top_logits.size(-1) <= 4096, "a row must have 1 to 4096 entries");
    TORCH_CHECK(top_index.scalar_type() == at::kInt || top_index.scalar_type() == at::kLong, "top_index must be int32 or int64");
    return {top_logits.contiguous(), top_index.contiguous(), (int)top_logits.size(-1), dtype_of(top_logits.scalar_type(), "top_logits"),
            top_index.scalar_type() == at::kInt ? 4 : 8};
}

// (loss, stats)
std::tuple<at::Tensor, at::Tensor> distill_topk(const at::Tensor& logits, const at::Tensor& top_logits, const at::Tensor& top_index,
                                                double temperature, int64_t reduction)
{
    not_recorded();
    const Rows z = as_rows(logits, "logits");
    const int dtype = dtype_of(logits.scalar_type(), "logits");
    TORCH_CHECK(logits.dim() >= 2, "logits must be (rows, columns)");
    TORCH_CHECK((float)temperature > 0 && (float)temperature * (float)temperature > 0 && std::isfinite((float)temperature * (float)temperature),
                "temperature must be positive, its square a float that is neither 0 nor infinite");
    TORCH_CHECK(z.rows >= 1, "logits have no rows");
    const Top top = as_top(z, logits, top_logits, top_index);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
    const auto options = logits.options().dtype(at::kFloat);
    const at::Tensor loss = reduction == GEO_SC_REDUCE_NONE ? row_scalars(logits) : at::empty({}, options), stats = at::empty({z.rows, 4}, options);
    size_t bytes = 0;
    check_status(geo_sc_distill_topk_workspace_size(z.rows, z.cols, &bytes), "workspace query");
    const at::Tensor workspace = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
    check_status(geo_sc_distill_topk(z.t.const_data_ptr(), dtype, z.stride, top.logits.const_data_ptr(), top.dtype, top.index.const_data_ptr(),
                                     top.index_bytes, z.rows, z.cols, top.top, (float)temperature, (int)reduction, loss.data_ptr<float>(),
                                     stats.data_ptr<float>(), workspace.data_ptr(), bytes, stream_of(logits)),
                 "distill_topk");
    return {loss, stats};
}

at::Tensor distill_topk_backward(const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& top_logits, const at::Tensor& top_index,
                                 double temperature, int64_t reduction, const at::Tensor& stats)
{
    not_recorded();
    const Rows z = as_rows(logits, "logits");
    const Top top = as_top(z, logits, top_logits, top_index);
    with(grad, "gradient", logits, "logits");
    TORCH_CHECK(grad.scalar_type() == at::kFloat && grad.numel() == (reduction == GEO_SC_REDUCE_NONE ? z.rows : 1),
                "gradient must have the shape and type of the loss");
    const at::Tensor g = grad.contiguous();
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
    const at::Tensor dz = at::empty(logits.sizes(), logits.options());
    check_status(geo_sc_distill_topk_backward(g.const_data_ptr<float>(), (int)reduction, z.t.const_data_ptr(),
                                              dtype_of(logits.scalar_type(), "logits"), z.stride, top.logits.const_data_ptr(), top.dtype,
                                              top.index.const_data_ptr(), top.index_bytes, z.rows, z.cols, top.top, (float)temperature,
                                              stats.const_data_ptr<float>(), dz.data_ptr(), stream_of(logits)),
                 "distill_topk backward");
    return once(dz, {grad});
}

// ---------------------------------------------------------------- autograd nodes
//
// In C++ like the calls themselves: of a training step on small layers the host's time is what counts, and the backward runs in
// the engine's thread without the interpreter.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

MaybeTensor maybe(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
at::Tensor undefined_or(const MaybeTensor& t) { return t ? *t : at::Tensor(); }

struct LinearQ8 : torch::autograd::Function<LinearQ8> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight)
    {
        const auto [q, scale, none] = quantize_rows(x, std::nullopt);
        const auto [wq, wscale, none2] = quantize_rows(weight, std::nullopt);
        ctx->save_for_backward({q, scale, wq, wscale});
        ctx->saved_data["x"] = x.scalar_type();
        ctx->saved_data["w"] = weight.scalar_type();
        return matmul_q8(q, scale, wq, wscale, x.scalar_type());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        std::optional<at::ScalarType> x, w;
        if (ctx->needs_input_grad(0)) x = ctx->saved_data["x"].toScalarType();
        if (ctx->needs_input_grad(1)) w = ctx->saved_data["w"].toScalarType();
        const auto [dx, dw] = matmul_q8_backward(grads[0], s[0], s[1], s[2], s[3], x, w);
        return {undefined_or(dx), undefined_or(dw)};
    }
};

// (q, scale, values, total); total is an output only where there is a residual
struct RmsNormQ8 : torch::autograd::Function<RmsNormQ8> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const MaybeTensor& residual, double eps,
                                 at::ScalarType values_type)
    {
        const auto [q, scale, total, values, rstd] = rms_norm_q8(x, weight, residual, eps, values_type, true);
        ctx->set_materialize_grads(false);
        const auto [first, second] = summands(x, residual, total);
        ctx->save_for_backward({first, second, weight, *rstd});
        ctx->mark_non_differentiable({q, scale});
        variable_list out = {q, scale, *values};
        if (residual) out.push_back(total);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const bool residual = grads.size() > 3;
        const auto [dx, dw] = rms_norm_q8_backward(maybe(grads[2]), residual ? maybe(grads[3]) : MaybeTensor(), s[0], s[1], s[2], s[3],
                                                   ctx->needs_input_grad(1));
        return {ctx->needs_input_grad(0) ? dx : at::Tensor(), undefined_or(dw), residual && ctx->needs_input_grad(2) ? dx : at::Tensor(),
                at::Tensor(), at::Tensor()};
    }
};

// (y, total); total is an output only where there is a residual
struct NormLinearQ8 : torch::autograd::Function<NormLinearQ8> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gain, const at::Tensor& weight,
                                 const MaybeTensor& residual, double eps)
    {
        const auto [q, scale, total, none, rstd] = rms_norm_q8(x, gain, residual, eps, std::nullopt, true);
        const auto [wq, wscale, none2] = quantize_rows(weight, std::nullopt);
        ctx->set_materialize_grads(false);
        const auto [first, second] = summands(x, residual, total);
        ctx->save_for_backward({q, scale, wq, wscale, first, second, gain, *rstd});
        ctx->saved_data["w"] = weight.scalar_type();
        variable_list out = {matmul_q8(q, scale, wq, wscale, x.scalar_type())};
        if (residual) out.push_back(total);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const bool residual = grads.size() > 1, need_gain = ctx->needs_input_grad(1);
        const bool through = ctx->needs_input_grad(0) || need_gain || (residual && ctx->needs_input_grad(3));
        MaybeTensor dn, dw, dgain;
        at::Tensor dx;
        if (grads[0].defined()) {
            std::optional<at::ScalarType> x, w;
            if (through) x = s[4].scalar_type();
            if (ctx->needs_input_grad(2)) w = ctx->saved_data["w"].toScalarType();
            std::tie(dn, dw) = matmul_q8_backward(grads[0], s[0], s[1], s[2], s[3], x, w);
        }
        if (through) std::tie(dx, dgain) = rms_norm_q8_backward(dn, residual ? maybe(grads[1]) : MaybeTensor(), s[4], s[5], s[6], s[7], need_gain);
        return {ctx->needs_input_grad(0) ? dx : at::Tensor(), undefined_or(dgain), undefined_or(dw),
                residual && ctx->needs_input_grad(3) ? dx : at::Tensor(), at::Tensor()};
    }
};

struct DistillTopK : torch::autograd::Function<DistillTopK> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& top_logits, const at::Tensor& top_index,
                              double temperature, int64_t reduction)
    {
        const auto [loss, stats] = distill_topk(logits, top_logits, top_index, temperature, reduction);
        ctx->save_for_backward({logits, top_logits, top_index, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        return {distill_topk_backward(grads[0], s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["reduction"].toInt(), s[3]),
                at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("quantize_rows", &quantize_rows, "rows in 8 bits: (q, scale, values or None)");
    m.def("rms_norm_q8", [](const at::Tensor& x, const at::Tensor& weight, const MaybeTensor& residual, double eps, std::optional<at::ScalarType> values) {
        const auto [q, scale, total, v, rstd] = rms_norm_q8(x, weight, residual, eps, values, false);
        return std::make_tuple(q, scale, total, v);
    }, "root-mean-square norm with 8-bit output: (q, scale, total, values or None)");
    m.def("rms_norm_q8_grad", [](const at::Tensor& x, const at::Tensor& weight, const MaybeTensor& residual, double eps, at::ScalarType values) {
        const variable_list out = RmsNormQ8::apply(x, weight, residual, eps, values);
        return std::make_tuple(out[0], out[1], residual ? out[3] : x, out[2]);
    }, "the same, values and total differentiable");
    m.def("matmul_q8", &matmul_q8, "product of 8-bit rows with a scale each");
    m.def("linear_q8", [](const at::Tensor& x, const at::Tensor& weight) { return LinearQ8::apply(x, weight); }, "product of x and weight rounded to 8-bit rows");
    m.def("norm_linear_q8", [](const at::Tensor& x, const at::Tensor& gain, const at::Tensor& weight, const MaybeTensor& residual, double eps) {
        const variable_list out = NormLinearQ8::apply(x, gain, weight, residual, eps);
        return std::make_tuple(out[0], residual ? out[1] : x);
    }, "the norm and the product: (y, total)");
    m.def("distill_topk", [](const at::Tensor& logits, const at::Tensor& top_logits, const at::Tensor& top_index, double temperature, int64_t reduction) {
        return DistillTopK::apply(logits, top_logits, top_index, temperature, reduction);
    }, "divergence from a teacher's top logits");
}
