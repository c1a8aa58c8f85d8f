// PyTorch module `sc_dense`: the dense 8-bit layers, the gated norm, the distillation loss and the AdamW step of libgeo_sc.so on tensors.  Checks, outputs
// and workspaces from the caching allocator, launch on PyTorch's current HIP stream.  In C++ because a single
// token's call is bound by its host time.
#include "sc_torch_common.h"

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>

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
                "the dense 8-bit layers, the gated norm, the distillation loss and the AdamW step cannot be traced");
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
        TORCH_CHECK(false, "the dense 8-bit layers, the gated norm and the distillation loss can be differentiated once only");
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

// ---------------------------------------------------------------- gated norm

// The description of a call, and the tensors that it points into.
struct Gated {
    Rows x, residual;
    at::Tensor weight;
    MaybeTensor post, gate, scale;
    geo_sc_gated_norm_desc desc;
};
Gated as_gated(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, const MaybeTensor& post, const MaybeTensor& gate,
               const MaybeTensor& scale, double eps)
{
    Gated g;
    g.x = as_rows(x, "x");
    const int dtype = dtype_of(x.scalar_type(), "x");
    with(residual, "residual", x, "x");
    TORCH_CHECK(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(), "residual must have the shape and type of x");
    g.residual = as_rows(residual, "residual");
    const auto per_channel = [&](const at::Tensor& t, const char* what) {
        with(t, what, x, "x");
        TORCH_CHECK(t.dim() == 1 && t.size(0) == g.x.cols, what, " must have the ", g.x.cols, " elements of a row of x");
        TORCH_CHECK(t.scalar_type() == x.scalar_type(), what, " must have the type of x");
        return t.contiguous();
    };
    g.weight = per_channel(weight, "weight");
    if (post) g.post = per_channel(*post, "post_weight");
    if (scale) g.scale = per_channel(*scale, "residual_scale");
    TORCH_CHECK(eps >= 0, "eps must not be negative");
    g.desc = {};
    g.desc.rows_per_gate = 1;
    if (gate && gate->dim() == 1) {
        g.gate = per_channel(*gate, "gate");
        g.desc.rows_per_gate = g.x.rows > 0 ? g.x.rows : 1;
    } else if (gate) {
        with(*gate, "gate", x, "x");
        TORCH_CHECK(gate->scalar_type() == x.scalar_type(), "gate must have the type of x");
        TORCH_CHECK(gate->dim() == x.dim() && gate->size(-1) == g.x.cols, "gate must have the ", g.x.cols,
                    " elements of a row of x, or the dimensions of x");
        // x's leading dimensions, then ones: rows that share a gate follow each other
        int64_t d = x.dim() - 2, shared = 1;
        for (; d >= 0 && gate->size(d) == 1; --d) shared *= x.size(d);
        for (; d >= 0; --d) TORCH_CHECK(gate->size(d) == x.size(d), "gate must have x's leading dimensions, then ones");
        g.gate = gate->contiguous();
        g.desc.rows_per_gate = shared > 0 ? shared : 1;
    }
    g.desc.struct_bytes = sizeof g.desc;
    g.desc.x = g.x.t.const_data_ptr();
    g.desc.residual = g.residual.t.const_data_ptr();
    g.desc.weight = g.weight.const_data_ptr();
    g.desc.post_weight = g.post ? g.post->const_data_ptr() : nullptr;
    g.desc.gate = g.gate ? g.gate->const_data_ptr() : nullptr;
    g.desc.residual_scale = g.scale ? g.scale->const_data_ptr() : nullptr;
    g.desc.rows = g.x.rows;
    g.desc.cols = g.x.cols;
    g.desc.x_stride = g.x.stride;
    g.desc.residual_stride = g.residual.stride;
    g.desc.eps = (float)eps;
    g.desc.dtype = dtype;
    return g;
}

// (out, total, rstd)
std::tuple<at::Tensor, at::Tensor, MaybeTensor> gated_norm(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight,
                                                           const MaybeTensor& post, const MaybeTensor& gate, const MaybeTensor& scale, double eps,
                                                           bool for_backward)
{
    not_recorded();
    const Gated g = as_gated(x, residual, weight, post, gate, scale, eps);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const at::Tensor out = at::empty(x.sizes(), x.options()), total = at::empty(x.sizes(), x.options());
    MaybeTensor rstd;
    if (for_backward) rstd = at::empty({g.x.rows, 2}, x.options().dtype(at::kFloat));
    check_status(geo_sc_gated_norm(&g.desc, out.data_ptr(), total.data_ptr(), (float*)data_of(rstd), stream_of(x)), "gated_norm");
    return {out, total, rstd};
}

// (q, scale, total, values, rstd)
std::tuple<at::Tensor, at::Tensor, at::Tensor, MaybeTensor, MaybeTensor> gated_norm_q8(const at::Tensor& x, const at::Tensor& residual,
                                                                                     const at::Tensor& weight, const MaybeTensor& post,
                                                                                     const MaybeTensor& gate, const MaybeTensor& scale, double eps,
                                                                                     std::optional<at::ScalarType> values_type, bool for_backward)
{
    not_recorded();
    Gated g = as_gated(x, residual, weight, post, gate, scale, eps);
    const int vtype = values_type ? dtype_of(*values_type, "values") : 0;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const at::Tensor q = empty_q(x.sizes(), x.options()), q_scale = row_scalars(x), total = at::empty(x.sizes(), x.options());
    MaybeTensor values;
    if (values_type) values = at::empty(x.sizes(), x.options().dtype(*values_type));
    MaybeTensor rstd;
    if (for_backward) rstd = at::empty({g.x.rows, 2}, x.options().dtype(at::kFloat));
    g.desc.rstd = (float*)data_of(rstd);
    check_status(geo_sc_gated_norm_q8(&g.desc, q.data_ptr<int8_t>(), (g.x.cols + 15) / 16 * 16, q_scale.data_ptr<float>(), total.data_ptr(),
                                      data_of(values), vtype, stream_of(x)),
                 "gated_norm_q8");
    return {q, q_scale, total, values, rstd};
}

struct GatedGradients {
    at::Tensor x, residual;
    MaybeTensor weight, post, gate, scale;
};
// `wanted`: of weight, post, gate, scale
GatedGradients gated_norm_backward(const at::Tensor& grad_out, const at::Tensor& grad_total, const at::Tensor& x, const at::Tensor& residual,
                                   const at::Tensor& weight, const MaybeTensor& post, const MaybeTensor& gate, const MaybeTensor& scale,
                                   double eps, const at::Tensor& rstd, const std::array<bool, 4>& wanted)
{
    not_recorded();
    const Gated g = as_gated(x, residual, weight, post, gate, scale, eps);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    GatedGradients d;
    const auto like = [](const at::Tensor& t, bool zero) { return zero ? at::zeros(t.sizes(), t.options()) : at::empty(t.sizes(), t.options()); };
    const bool none = g.x.rows == 0 || (!grad_out.defined() && !grad_total.defined());
    d.x = like(x, none);
    d.residual = like(residual, none);
    if (wanted[0]) d.weight = like(g.weight, none);
    if (wanted[1] && g.post) d.post = like(*g.post, none);
    if (wanted[2] && g.gate) d.gate = like(*g.gate, none);
    if (wanted[3] && g.scale) d.scale = like(*g.scale, none);
    if (none) return d;
    Rows out = {}, total = {};
    out = as_rows(grad_out.defined() ? grad_out.to(x.scalar_type()) : at::zeros(x.sizes(), x.options()), "gradient");
    if (grad_total.defined()) total = as_rows(grad_total.to(x.scalar_type()), "gradient");
    size_t bytes = 0;
    check_status(geo_sc_gated_norm_backward_workspace_size(g.x.rows, g.x.cols, &bytes), "workspace query");
    const at::Tensor workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check_status(geo_sc_gated_norm_backward(&g.desc, out.t.const_data_ptr(), out.stride, grad_total.defined() ? total.t.const_data_ptr() : nullptr,
                                            total.stride, rstd.const_data_ptr<float>(), d.x.data_ptr(), d.residual.data_ptr(), data_of(d.weight),
                                            data_of(d.post), data_of(d.gate), data_of(d.scale), workspace.data_ptr(), bytes, stream_of(x)),
                 "gated_norm backward");
    for (const MaybeTensor& t : {MaybeTensor(d.x), MaybeTensor(d.residual), d.weight, d.post, d.gate, d.scale})
        if (t) once(*t, {grad_out, grad_total});
    return d;
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

// What follows a product: bias, activation, residual, and whether the backward will ask for the activation's slope.
struct After {
    MaybeTensor bias, residual;
    int activation = GEO_SC_ACT_NONE;
    bool keep_slope = false;
    at::Tensor slope;   // what came of it
    bool any() const { return bias || residual || activation != GEO_SC_ACT_NONE; }
};
int activation_of(const std::optional<std::string>& name)
{
    if (!name) return GEO_SC_ACT_NONE;
    if (*name == "relu") return GEO_SC_ACT_RELU;
    if (*name == "gelu") return GEO_SC_ACT_GELU;
    if (*name == "silu") return GEO_SC_ACT_SILU;
    TORCH_CHECK(false, "activation must be None, 'relu', 'gelu' or 'silu', got '", *name, "'");
}

at::Tensor matmul_q8(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& wq, const at::Tensor& wscale, at::ScalarType type, After& after)
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
    geo_sc_q8_epilogue e = {};
    at::Tensor bias;
    Rows residual;
    if (after.bias) {
        with(*after.bias, "bias", q, "q");
        TORCH_CHECK(after.bias->dim() == 1 && after.bias->size(0) == w.r.rows, "bias must have the ", w.r.rows, " elements of a row of the product");
        e.bias_dtype = dtype_of(after.bias->scalar_type(), "bias");
        bias = after.bias->contiguous();
        e.bias = bias.const_data_ptr();
    }
    if (after.residual) {
        with(*after.residual, "residual", q, "q");
        TORCH_CHECK(after.residual->sizes() == at::IntArrayRef(sizes) && after.residual->scalar_type() == type,
                    "residual must have the shape and type of the product");
    }
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    const at::Tensor y = at::empty(sizes, q.options().dtype(type));
    if (after.keep_slope) {
        // a relu's slope is 0 or 1; others in fp16 are off by an eighth of what bf16 rounds by, and beside fp16's own rounding that would
        // show (gradients of 4000 x 500 fp16 1.5 times as far off)
        const at::ScalarType kept = after.activation == GEO_SC_ACT_RELU ? at::kByte : type == at::kBFloat16 ? at::kHalf : at::kFloat;
        after.slope = at::empty({x.r.rows, w.r.rows}, q.options().dtype(kept));
        e.slope_dtype = kept == at::kByte ? GEO_SC_U8 : dtype_of(kept, "slope");
    }
    if (y.numel() == 0) return y;
    if (after.residual) {
        residual = as_rows(*after.residual, "residual");
        e.residual = residual.t.const_data_ptr();
        e.residual_stride = residual.stride;
    }
    size_t bytes = 0;
    check_status(geo_sc_matmul_q8_workspace_size(x.r.t.const_data_ptr<int8_t>(), x.r.stride, w.r.t.const_data_ptr<int8_t>(),
                                                 w.r.stride, x.r.rows, w.r.rows, x.r.cols, &bytes), "workspace query");
    MaybeTensor workspace;
    if (bytes) workspace = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    if (after.any()) {
        e.struct_bytes = sizeof e;
        e.activation = after.activation;
        e.slope = after.keep_slope ? after.slope.data_ptr() : nullptr;
        check_status(geo_sc_matmul_q8_epilogue(x.r.t.const_data_ptr<int8_t>(), x.r.stride, x.scale.const_data_ptr<float>(),
                                               w.r.t.const_data_ptr<int8_t>(), w.r.stride, w.scale.const_data_ptr<float>(), x.r.rows, w.r.rows,
                                               x.r.cols, &e, y.data_ptr(), dtype, data_of(workspace), bytes, stream_of(q)),
                     "matmul_q8");
        return y;
    }
    check_status(geo_sc_matmul_q8(x.r.t.const_data_ptr<int8_t>(), x.r.stride, x.scale.const_data_ptr<float>(), w.r.t.const_data_ptr<int8_t>(),
                                  w.r.stride, w.scale.const_data_ptr<float>(), x.r.rows, w.r.rows, x.r.cols, y.data_ptr(), dtype,
                                  data_of(workspace), bytes, stream_of(q)),
                 "matmul_q8");
    return y;
}
at::Tensor matmul_q8(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& wq, const at::Tensor& wscale, at::ScalarType type)
{
    After none;
    return matmul_q8(q, scale, wq, wscale, type, none);
}

struct ProductGradients {
    MaybeTensor x, w, bias;
};
// `slope`: of the activation, or undefined; y_type is the product's type then
ProductGradients matmul_q8_backward(const at::Tensor& grad, const at::Tensor& q, const at::Tensor& scale, const at::Tensor& wq,
                                    const at::Tensor& wscale, std::optional<at::ScalarType> dx_type, std::optional<at::ScalarType> dw_type,
                                    const at::Tensor& slope = {}, std::optional<at::ScalarType> dbias_type = std::nullopt)
{
    not_recorded();
    const Q8 x = as_q8(q, scale, "q"), w = as_q8(wq, wscale, "weight_q");
    if (w.r.rows == 0 && grad.numel() == 0) {   // no columns: sums of nothing
        on_gpu(grad, "gradient");
        return {dx_type ? MaybeTensor(at::zeros(q.sizes(), q.options().dtype(*dx_type))) : MaybeTensor(),
                dw_type ? MaybeTensor(at::empty(wq.sizes(), q.options().dtype(*dw_type))) : MaybeTensor(),
                dbias_type ? MaybeTensor(at::empty({0}, q.options().dtype(*dbias_type))) : MaybeTensor()};
    }
    Rows g = as_rows(grad, "gradient");
    if (g.rows > 1 && g.stride && g.stride < g.cols) g = as_rows(grad.contiguous(), "gradient");   // (rows that overlap)
    with(grad, "gradient", q, "q");
    TORCH_CHECK(x.r.cols == w.r.cols && g.rows == x.r.rows && g.cols == w.r.rows, "gradient must have the shape of the product");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    MaybeTensor dx, dw, dbias;
    if (dx_type) dx = at::empty(q.sizes(), q.options().dtype(*dx_type));
    if (dw_type) dw = at::empty(wq.sizes(), q.options().dtype(*dw_type));
    if (dbias_type) dbias = at::empty({g.cols}, q.options().dtype(*dbias_type));
    if (g.rows == 0 && dw) dw->zero_();
    if (g.rows == 0 && dbias) dbias->zero_();
    if (g.rows == 0 || (!dx && !dw && !dbias)) return {dx, dw, dbias};
    const int grad_type = dtype_of(g.t.scalar_type(), "gradient");
    size_t bytes = 0;
    check_status(geo_sc_matmul_q8_epilogue_backward_workspace_size(g.rows, g.cols, x.r.cols, grad_type, dx.has_value(), dw.has_value(),
                                                                   dbias.has_value(), &bytes),
                 "workspace query");
    const at::Tensor workspace = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check_status(geo_sc_matmul_q8_epilogue_backward(g.t.const_data_ptr(), grad_type, g.stride, slope.defined() ? slope.const_data_ptr() : nullptr,
                                                    !slope.defined() ? 0 : slope.scalar_type() == at::kByte ? GEO_SC_U8 : dtype_of(slope.scalar_type(), "slope"),
                                                    x.r.t.const_data_ptr<int8_t>(), x.r.stride, x.scale.const_data_ptr<float>(),
                                                    w.r.t.const_data_ptr<int8_t>(), w.r.stride, w.scale.const_data_ptr<float>(), g.rows, g.cols,
                                                    x.r.cols, data_of(dx), dx ? dtype_of(*dx_type, "dx") : 0, data_of(dw),
                                                    dw ? dtype_of(*dw_type, "dw") : 0, data_of(dbias), dbias ? dtype_of(*dbias_type, "dbias") : 0,
                                                    workspace.data_ptr(), bytes, stream_of(q)),
                 "matmul_q8 backward");
    for (const MaybeTensor& d : {dx, dw, dbias})
        if (d) once(*d, {grad});
    return {dx, dw, dbias};
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

// ---------------------------------------------------------------- AdamW

using Tensors = std::vector<at::Tensor>;
using MaybeTensors = std::optional<Tensors>;

// What one of the lists of a step must be: on the GPU of the first parameter, side by side, of the parameter's element count (of its
// blocks'), of the type or types named.
// `param`: or NULL; what goes with it element by element has its shape.
void in_step(const at::Tensor& t, const char* what, const at::Tensor& first, int64_t elements, std::initializer_list<at::ScalarType> types,
             const at::Tensor* param = nullptr)
{
    with(t, what, first, "params");
    TORCH_CHECK(t.is_contiguous(), what, " must be contiguous");
    if (!param || t.sizes() != param->sizes()) {
        TORCH_CHECK(t.numel() == elements, what, " must have ", elements, " elements, got ", t.numel());
        TORCH_CHECK(!param, what, " must have the shape of its parameter, ", param->sizes(), ", got ", t.sizes());
    }
    for (const at::ScalarType type : types)
        if (t.scalar_type() == type) return;
    TORCH_CHECK(false, what, " must not be ", t.scalar_type());
}

constexpr int64_t kStateBlock = 256;

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& exp_avg, const Tensors& exp_avg_sq, int64_t step,
                const MaybeTensor& device_step, double lr, double beta1, double beta2, double eps, double weight_decay, double grad_scale,
                const MaybeTensors& avg_scales, const MaybeTensors& sq_scales, const MaybeTensors& copies,
                const std::optional<std::vector<MaybeTensor>>& clamped, double lo, double hi)
{
    not_recorded();
    const size_t n = params.size();
    TORCH_CHECK(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n && (!avg_scales || avg_scales->size() == n) &&
                    (!sq_scales || sq_scales->size() == n) && (!copies || copies->size() == n) && (!clamped || clamped->size() == n),
                "the lists of a step must be of one length");
    TORCH_CHECK(lr >= 0 && eps >= 0 && weight_decay >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && lo <= hi,
                "lr, eps and weight_decay must not be negative, the betas must be in [0, 1), the bounds in order");
    TORCH_CHECK(device_step || step >= 1, "the number of a step is 1 or more");
    if (!n) return;
    const at::Tensor& first = params[0];
    const bool eight = avg_scales.has_value();
    if (device_step) in_step(*device_step, "step", first, 1, {at::kLong});
    // Tensors of the same types go into one call; no writer meets another.
    typedef std::array<int, 3> Types;
    std::vector<std::pair<Types, std::vector<geo_sc_adamw_tensor>>> calls;
    std::vector<std::pair<const char*, const char*>> written;   // begin, end
    written.reserve(n * 7);
    const auto write = [&](const at::Tensor& t) {
        TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), "an inference tensor is written to in inference mode only");
        void* p = t.data_ptr();
        if (t.numel()) written.emplace_back((const char*)p, (const char*)p + t.nbytes());
        return p;
    };
    for (size_t i = 0; i < n; ++i) {
        const int64_t elements = params[i].numel(), blocks = (elements + kStateBlock - 1) / kStateBlock;
        geo_sc_adamw_tensor t = {};
        t.elements = elements;
        in_step(params[i], "params", first, elements, {at::kFloat, at::kBFloat16, at::kHalf});
        in_step(grads[i], "grads", first, elements, {at::kFloat, at::kBFloat16, at::kHalf}, &params[i]);
        t.param = write(params[i]);
        t.grad = grads[i].const_data_ptr();
        for (const auto& [state, scales, what, codes, scale] : {std::make_tuple(&exp_avg, &avg_scales, "exp_avg", &t.exp_avg, &t.avg_scale),
                                                                std::make_tuple(&exp_avg_sq, &sq_scales, "exp_avg_sq", &t.exp_avg_sq, &t.sq_scale)}) {
            in_step((*state)[i], what, first, elements, {eight ? at::kFloat8_e4m3fn : at::kFloat}, &params[i]);
            *codes = write((*state)[i]);
            if (!eight) continue;
            in_step((**scales)[i], "scales", first, blocks, {at::kFloat8_e8m0fnu});
            *scale = (uint8_t*)write((**scales)[i]);
        }
        if (copies) {
            in_step((*copies)[i], "copies", first, elements, {at::kFloat, at::kBFloat16, at::kHalf}, &params[i]);
            t.copy = write((*copies)[i]);
        }
        if (clamped && (*clamped)[i]) {
            in_step(*(*clamped)[i], "clamped", first, elements, {at::kFloat}, &params[i]);
            t.clamped = (float*)write(*(*clamped)[i]);
        }
        const Types types = {dtype_of(params[i].scalar_type(), "params"), dtype_of(grads[i].scalar_type(), "grads"),
                             copies ? dtype_of((*copies)[i].scalar_type(), "copies") : 0};
        size_t k = 0;
        while (k < calls.size() && calls[k].first != types) ++k;
        if (k == calls.size()) {
            calls.emplace_back(types, std::vector<geo_sc_adamw_tensor>());
            calls[k].second.reserve(n - i);
        }
        calls[k].second.push_back(t);
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i) TORCH_CHECK(written[i - 1].second <= written[i].first, "a step writes no memory twice");
    for (const at::Tensor& g : grads) {   // (one gradient may serve several parameters, but not be written over on the way)
        const char* begin = (const char*)g.const_data_ptr();
        const auto above = std::lower_bound(written.begin(), written.end(), begin + g.nbytes(),
                                            [](const auto& range, const char* end) { return range.first < end; });   // the first range behind it
        TORCH_CHECK(g.numel() == 0 || above == written.begin() || (above - 1)->second <= begin, "a step writes none of its gradients");
    }
    TORCH_CHECK(!device_step || calls.size() == 1, "a step that is counted on the GPU takes tensors of the same types");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(first.device());
    at::Tensor workspace;
    if (device_step) workspace = at::empty({16}, first.options().dtype(at::kByte));
    for (const auto& [types, tensors] : calls) {
        geo_sc_adamw_options o = {};
        o.struct_bytes = sizeof o;
        o.param_dtype = types[0];
        o.grad_dtype = types[1];
        o.copy_dtype = types[2];
        o.state_bits = eight ? 8 : 32;
        o.lr = lr;
        o.beta1 = beta1;
        o.beta2 = beta2;
        o.eps = eps;
        o.weight_decay = weight_decay;
        o.grad_scale = grad_scale;
        o.lo = (float)lo;
        o.hi = (float)hi;
        o.step = step;
        o.device_step = device_step ? device_step->data_ptr<int64_t>() : nullptr;
        check_status(geo_sc_adamw((int)tensors.size(), tensors.data(), &o, device_step ? workspace.data_ptr() : nullptr, device_step ? 16 : 0,
                                  stream_of(first)),
                     "adamw_step");
    }
    // (for whoever watches a tensor's version: autograd, prepared weights)
    const auto changed = [](const at::Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); };
    for (const Tensors* list : {&params, &exp_avg, &exp_avg_sq})
        for (const at::Tensor& t : *list) changed(t);
    for (const MaybeTensors* list : {&avg_scales, &sq_scales, &copies})
        if (*list)
            for (const at::Tensor& t : **list) changed(t);
    if (clamped)
        for (const MaybeTensor& t : *clamped)
            if (t) changed(*t);
    if (device_step) changed(*device_step);
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
        const ProductGradients d = matmul_q8_backward(grads[0], s[0], s[1], s[2], s[3], x, w);
        return {undefined_or(d.x), undefined_or(d.w)};
    }
};

// the same with an epilogue
struct LinearQ8Epilogue : torch::autograd::Function<LinearQ8Epilogue> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
                              int64_t activation, bool keep_slope)
    {
        const auto [q, scale, none] = quantize_rows(x, std::nullopt);
        const auto [wq, wscale, none2] = quantize_rows(weight, std::nullopt);
        After after;
        after.bias = bias;
        after.residual = residual;
        after.activation = (int)activation;
        after.keep_slope = keep_slope;
        const at::Tensor y = matmul_q8(q, scale, wq, wscale, x.scalar_type(), after);
        ctx->save_for_backward({q, scale, wq, wscale, after.slope});
        ctx->saved_data["x"] = x.scalar_type();
        ctx->saved_data["w"] = weight.scalar_type();
        if (bias) ctx->saved_data["bias"] = bias->scalar_type();
        ctx->saved_data["residual"] = residual.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const bool has_bias = ctx->saved_data.count("bias");
        std::optional<at::ScalarType> x, w, bias;
        if (ctx->needs_input_grad(0)) x = ctx->saved_data["x"].toScalarType();
        if (ctx->needs_input_grad(1)) w = ctx->saved_data["w"].toScalarType();
        if (has_bias && ctx->needs_input_grad(2)) bias = ctx->saved_data["bias"].toScalarType();
        ProductGradients d;
        if (x || w || bias) d = matmul_q8_backward(grads[0], s[0], s[1], s[2], s[3], x, w, s[4], bias);
        return {undefined_or(d.x), undefined_or(d.w), undefined_or(d.bias), ctx->saved_data["residual"].toBool() ? grads[0] : at::Tensor(),
                at::Tensor(), at::Tensor()};
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
                                 const MaybeTensor& residual, double eps, const MaybeTensor& bias, int64_t activation, bool keep_slope)
    {
        const auto [q, scale, total, none, rstd] = rms_norm_q8(x, gain, residual, eps, std::nullopt, true);
        const auto [wq, wscale, none2] = quantize_rows(weight, std::nullopt);
        ctx->set_materialize_grads(false);
        const auto [first, second] = summands(x, residual, total);
        After after;
        after.bias = bias;
        after.activation = (int)activation;
        after.keep_slope = keep_slope;
        variable_list out = {matmul_q8(q, scale, wq, wscale, x.scalar_type(), after)};
        ctx->save_for_backward({q, scale, wq, wscale, first, second, gain, *rstd, after.slope});
        ctx->saved_data["w"] = weight.scalar_type();
        if (bias) ctx->saved_data["bias"] = bias->scalar_type();
        if (residual) out.push_back(total);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const bool residual = grads.size() > 1, need_gain = ctx->needs_input_grad(1);
        const bool through = ctx->needs_input_grad(0) || need_gain || (residual && ctx->needs_input_grad(3));
        const bool need_bias = ctx->saved_data.count("bias") && ctx->needs_input_grad(3 + residual);
        ProductGradients d;
        MaybeTensor dgain;
        at::Tensor dx;
        if (grads[0].defined()) {
            std::optional<at::ScalarType> x, w, bias;
            if (through) x = s[4].scalar_type();
            if (ctx->needs_input_grad(2)) w = ctx->saved_data["w"].toScalarType();
            if (need_bias) bias = ctx->saved_data["bias"].toScalarType();
            d = matmul_q8_backward(grads[0], s[0], s[1], s[2], s[3], x, w, s[8], bias);
        }
        if (through) std::tie(dx, dgain) = rms_norm_q8_backward(d.x, residual ? maybe(grads[1]) : MaybeTensor(), s[4], s[5], s[6], s[7], need_gain);
        return {ctx->needs_input_grad(0) ? dx : at::Tensor(), undefined_or(dgain), undefined_or(d.w),
                residual && ctx->needs_input_grad(3) ? dx : at::Tensor(), at::Tensor(), undefined_or(d.bias), at::Tensor(), at::Tensor()};
    }
};

// Which of weight (at `at` of the inputs) and of `around`, which follow each other, the gradients are wanted of: inputs are counted
// without those that are None.
std::array<bool, 4> wanted_of(AutogradContext* ctx, size_t weight, size_t at, const at::Tensor* around)
{
    std::array<bool, 4> wanted = {ctx->needs_input_grad(weight), false, false, false};
    for (size_t i = 0; i < 3; ++i)
        if (around[i].defined()) wanted[1 + i] = ctx->needs_input_grad(at++);
    return wanted;
}

// (out, total)
struct GatedNorm : torch::autograd::Function<GatedNorm> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight,
                                 const MaybeTensor& post, const MaybeTensor& gate, const MaybeTensor& scale, double eps)
    {
        const auto [out, total, rstd] = gated_norm(x, residual, weight, post, gate, scale, eps, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, residual, weight, undefined_or(post), undefined_or(gate), undefined_or(scale), *rstd});
        ctx->saved_data["eps"] = eps;
        return {out, total};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const auto wanted = wanted_of(ctx, 2, 3, &s[3]);
        const GatedGradients d = gated_norm_backward(grads[0], grads[1], s[0], s[1], s[2], maybe(s[3]), maybe(s[4]), maybe(s[5]),
                                                     ctx->saved_data["eps"].toDouble(), s[6], wanted);
        return {ctx->needs_input_grad(0) ? d.x : at::Tensor(), ctx->needs_input_grad(1) ? d.residual : at::Tensor(), undefined_or(d.weight),
                undefined_or(d.post), undefined_or(d.gate), undefined_or(d.scale), at::Tensor()};
    }
};

// The gated norm with 8-bit output and the product: (y, total)
struct GatedNormLinearQ8 : torch::autograd::Function<GatedNormLinearQ8> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual, const at::Tensor& gain, const at::Tensor& weight,
                                 const MaybeTensor& post, const MaybeTensor& gate, const MaybeTensor& scale, const MaybeTensor& bias, double eps,
                                 int64_t activation, bool keep_slope)
    {
        const auto [q, q_scale, total, none, rstd] = gated_norm_q8(x, residual, gain, post, gate, scale, eps, std::nullopt, true);
        const auto [wq, wscale, none2] = quantize_rows(weight, std::nullopt);
        ctx->set_materialize_grads(false);
        After after;
        after.bias = bias;
        after.activation = (int)activation;
        after.keep_slope = keep_slope;
        const at::Tensor y = matmul_q8(q, q_scale, wq, wscale, x.scalar_type(), after);
        ctx->save_for_backward({q, q_scale, wq, wscale, x, residual, gain, undefined_or(post), undefined_or(gate), undefined_or(scale), *rstd, after.slope});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["w"] = weight.scalar_type();
        if (bias) ctx->saved_data["bias"] = bias->scalar_type();
        return {y, total};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const size_t at_bias = 4 + s[7].defined() + s[8].defined() + s[9].defined();
        const auto wanted = wanted_of(ctx, 2, 4, &s[7]);
        const bool through = ctx->needs_input_grad(0) || ctx->needs_input_grad(1) || wanted[0] || wanted[1] || wanted[2] || wanted[3];
        ProductGradients d;
        if (grads[0].defined()) {
            std::optional<at::ScalarType> x, w, bias;
            if (through) x = s[4].scalar_type();
            if (ctx->needs_input_grad(3)) w = ctx->saved_data["w"].toScalarType();
            if (ctx->saved_data.count("bias") && ctx->needs_input_grad(at_bias)) bias = ctx->saved_data["bias"].toScalarType();
            if (x || w || bias) d = matmul_q8_backward(grads[0], s[0], s[1], s[2], s[3], x, w, s[11], bias);
        }
        GatedGradients n;
        if (through)
            n = gated_norm_backward(undefined_or(d.x), grads[1], s[4], s[5], s[6], maybe(s[7]), maybe(s[8]), maybe(s[9]),
                                    ctx->saved_data["eps"].toDouble(), s[10], wanted);
        return {ctx->needs_input_grad(0) ? n.x : at::Tensor(), ctx->needs_input_grad(1) ? n.residual : at::Tensor(), undefined_or(n.weight),
                undefined_or(d.w), undefined_or(n.post), undefined_or(n.gate), undefined_or(n.scale), undefined_or(d.bias), at::Tensor(),
                at::Tensor(), at::Tensor()};
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
    m.def("matmul_q8", py::overload_cast<const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::ScalarType>(&matmul_q8),
          "product of 8-bit rows with a scale each");
    m.def("matmul_q8_epilogue", [](const at::Tensor& q, const at::Tensor& scale, const at::Tensor& wq, const at::Tensor& wscale, at::ScalarType type,
                                   const MaybeTensor& bias, const std::optional<std::string>& activation, const MaybeTensor& residual) {
        After after;
        after.bias = bias;
        after.residual = residual;
        after.activation = activation_of(activation);
        return matmul_q8(q, scale, wq, wscale, type, after);
    }, "the same with bias, activation and residual");
    m.def("linear_q8_epilogue", [](const at::Tensor& x, const at::Tensor& weight, const MaybeTensor& bias, const std::optional<std::string>& activation,
                                   const MaybeTensor& residual) {
        const int kind = activation_of(activation);
        // (the slope is for the gradients of all but the residual)
        const bool keep = kind != GEO_SC_ACT_NONE && at::GradMode::is_enabled() &&
                          (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()));
        return LinearQ8Epilogue::apply(x, weight, bias, residual, kind, keep);
    }, "product of x and weight rounded to 8-bit rows, with bias, activation and residual");
    m.def("linear_q8", [](const at::Tensor& x, const at::Tensor& weight) { return LinearQ8::apply(x, weight); }, "product of x and weight rounded to 8-bit rows");
    m.def("norm_linear_q8", [](const at::Tensor& x, const at::Tensor& gain, const at::Tensor& weight, const MaybeTensor& residual, double eps,
                               const MaybeTensor& bias, const std::optional<std::string>& activation) {
        const int kind = activation_of(activation);
        const bool keep = kind != GEO_SC_ACT_NONE && at::GradMode::is_enabled() &&
                          (x.requires_grad() || gain.requires_grad() || weight.requires_grad() || (residual && residual->requires_grad()) ||
                           (bias && bias->requires_grad()));
        const variable_list out = NormLinearQ8::apply(x, gain, weight, residual, eps, bias, kind, keep);
        return std::make_tuple(out[0], residual ? out[1] : x);
    }, "the norm and the product: (y, total)");
    m.def("gated_norm", [](const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, const MaybeTensor& post, const MaybeTensor& gate,
                           const MaybeTensor& scale, double eps, bool differentiable) {
        if (differentiable) {
            const variable_list out = GatedNorm::apply(x, residual, weight, post, gate, scale, eps);
            return std::make_tuple(out[0], out[1]);
        }
        const auto [out, total, none] = gated_norm(x, residual, weight, post, gate, scale, eps, false);
        return std::make_tuple(out, total);
    }, "norm behind a block, gate, scaled residual and the next norm: (out, total)");
    m.def("gated_norm_q8", [](const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, const MaybeTensor& post, const MaybeTensor& gate,
                              const MaybeTensor& scale, double eps, std::optional<at::ScalarType> values) {
        const auto [q, q_scale, total, v, none] = gated_norm_q8(x, residual, weight, post, gate, scale, eps, values, false);
        return std::make_tuple(q, q_scale, total, v);
    }, "the same with 8-bit output: (q, scale, total, values or None)");
    m.def("gated_norm_linear_q8", [](const at::Tensor& x, const at::Tensor& residual, const at::Tensor& gain, const at::Tensor& weight, const MaybeTensor& post,
                                     const MaybeTensor& gate, const MaybeTensor& scale, double eps, const MaybeTensor& bias,
                                     const std::optional<std::string>& activation) {
        const int kind = activation_of(activation);
        const auto wants = [](const MaybeTensor& t) { return t && t->requires_grad(); };
        const bool keep = kind != GEO_SC_ACT_NONE && at::GradMode::is_enabled() &&
                          (x.requires_grad() || residual.requires_grad() || gain.requires_grad() || weight.requires_grad() || wants(post) ||
                           wants(gate) || wants(scale) || wants(bias));
        const variable_list out = GatedNormLinearQ8::apply(x, residual, gain, weight, post, gate, scale, bias, eps, kind, keep);
        return std::make_tuple(out[0], out[1]);
    }, "the gated norm with 8-bit output and the product: (y, total)");
    m.def("adamw_step", &adamw_step, "one AdamW step on lists of tensors");
    m.def("distill_topk", [](const at::Tensor& logits, const at::Tensor& top_logits, const at::Tensor& top_index, double temperature, int64_t reduction) {
        return DistillTopK::apply(logits, top_logits, top_index, temperature, reduction);
    }, "divergence from a teacher's top logits");
}
