// torch ops of the feed-forward half of a layer: mxrec::layer_norm, mxrec::gated_linear (both with autograd) and
// mxrec::activation_pack8 / activation_unpack8.  Argument checks, output allocation and the calls of the C ABI in hstu_ffn.h;
// no counterpart in the reference.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <cstring>

#include "hstu_ffn.h"

namespace mxrec_ffn {

static int32_t type_code(at::ScalarType t, const char* op, const char* name) {
    switch (t) {
        case at::kFloat: return HSTU_F32;
        case at::kHalf: return HSTU_F16;
        case at::kBFloat16: return HSTU_BF16;
        default: TORCH_CHECK(false, op, ": ", name, " dtype expect float32, float16 or bfloat16, but get ", t);
    }
}

// The tensors of one call: all on the GPU that the first one is on.  The device is made current, the work goes to that
// device's current stream.
static void check_devices(const char* op, std::initializer_list<const at::Tensor*> ts) {
    const at::Tensor& first = **ts.begin();
    for (const at::Tensor* t : ts)
        if (t->defined()) TORCH_CHECK(t->device() == first.device(), op, ": all tensors must be on one device, but get ", t->device(), " and ", first.device());
    TORCH_CHECK(first.is_cuda(), op, " has no CPU implementation: move the tensors to the MI355X (device 'cuda')");
}

// [rows, last dim] with unit stride along the last dim: a view where the layout allows one (row strides stay), else a copy
static at::Tensor rows_of(const at::Tensor& t) {
    const int64_t c = t.size(-1);
    at::Tensor r = t.dim() == 2 ? t : t.numel() == 0 ? at::empty({t.numel() / (c ? c : 1), c}, t.options()) : t.reshape({-1, c});
    if (c > 1 && r.stride(1) != 1) r = r.contiguous();
    return r;
}
// rows of a tensor: product of all sizes but the last (also where the last dim or the tensor is empty)
static int64_t row_count(const at::Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < t.dim(); i++) n *= t.size(i);
    return n;
}

struct Launch {   // current device and stream of a call
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
    explicit Launch(const at::Tensor& t) : guard(t.device()) {}
    void* stream() const { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
};

// an optional tensor argument; undefined where it is missing
static at::Tensor value(const c10::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }

// Forward-mode derivatives are not implemented, and a result without a tangent counts as a constant: inputs that carry one are refused
// (not where forward mode is switched off, as in the forward of a caller's own autograd function).
static void no_tangents(const char* op, std::initializer_list<const at::Tensor*> ts) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const at::Tensor* t : ts) TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op, ": forward-mode derivatives are not supported (an input carries a tangent)");
}
static void no_double_backward(const char* op, const at::Tensor& grad) {
    TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the backward is not differentiable (called with create_graph=True)");
    no_tangents(op, {&grad});
}

// ---- layer_norm --------------------------------------------------------------------------------------------------------
static const char* LN = "mxrec::layer_norm";

static void ln_check(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, double eps) {
    TORCH_CHECK(x.defined() && x.dim() >= 1, LN, ": x must have at least 1 dimension");
    type_code(x.scalar_type(), LN, "x");
    const int64_t c = x.size(-1);
    TORCH_CHECK(c >= 1 && c <= HSTU_LN_MAX_COLS, LN, ": the last dimension of x must in range:[1,", HSTU_LN_MAX_COLS, "], but get ", c);
    const at::Tensor* ps[2] = {&weight, &bias};
    const char* names[2] = {"weight", "bias"};
    for (int i = 0; i < 2; i++) {
        const at::Tensor& p = *ps[i];
        if (!p.defined()) continue;
        TORCH_CHECK(p.dim() == 1 && p.size(0) == c, LN, ": ", names[i], " must be 1D with the size of the last dimension of x (", c, "), but get ", p.sizes());
        TORCH_CHECK(p.scalar_type() == x.scalar_type() || p.scalar_type() == at::kFloat, LN, ": ", names[i], " dtype expect ", x.scalar_type(),
                    " or float32, but get ", p.scalar_type());
    }
    if (weight.defined() && bias.defined())
        TORCH_CHECK(weight.scalar_type() == bias.scalar_type(), LN, ": weight and bias must have one dtype, but get ", weight.scalar_type(), " and ", bias.scalar_type());
    // as the kernel sees it: in single precision
    TORCH_CHECK((float)eps > 0.f && std::isfinite((float)eps), LN, ": eps must be positive and finite, but get ", eps);
}

static at::ScalarType ln_param_type(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias) {
    return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
}

// {y} or {y, mean, rstd}
static std::vector<at::Tensor> ln_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, double eps, bool stats) {
    ln_check(x, weight, bias, eps);
    no_tangents(LN, {&x, &weight, &bias});
    check_devices(LN, {&x, &weight, &bias});
    Launch launch(x);
    const at::Tensor xr = rows_of(x), w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    const int64_t rows = row_count(x);
    std::vector<at::Tensor> outs{at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous))};
    hstu_layer_norm_params p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.dtype = type_code(x.scalar_type(), LN, "x");
    p.param_dtype = type_code(ln_param_type(x, weight, bias), LN, "weight");
    p.cols = (int32_t)x.size(-1);
    p.rows = rows;
    p.x_stride = rows > 1 ? xr.stride(0) : p.cols;
    p.eps = (float)eps;
    p.x = xr.const_data_ptr();
    p.weight = w.defined() ? w.const_data_ptr() : nullptr;
    p.bias = b.defined() ? b.const_data_ptr() : nullptr;
    p.y = outs[0].data_ptr();
    if (stats) {
        auto shape = x.sizes().vec();
        shape.pop_back();
        for (int i = 0; i < 2; i++) outs.push_back(at::empty(shape, x.options().dtype(at::kFloat)));
        p.mean = rows ? outs[1].data_ptr<float>() : nullptr;
        p.rstd = rows ? outs[2].data_ptr<float>() : nullptr;
    }
    const int rc = hstu_hip_layer_norm(&p, launch.stream());
    TORCH_CHECK(rc == HSTU_OK, LN, ": ", hstu_hip_last_error());
    return outs;
}

// {d_x, d_weight, d_bias}, undefined where not wanted; the parameter gradients in grad_type
static std::vector<at::Tensor> ln_backward(const at::Tensor& d_y, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& mean,
                                           const at::Tensor& rstd, at::ScalarType param_type, at::ScalarType grad_type, bool want_x, bool want_w, bool want_b) {
    check_devices(LN, {&x, &weight, &d_y, &mean, &rstd});
    Launch launch(x);
    const int64_t rows = row_count(x), c = x.size(-1);
    const at::Tensor xr = rows_of(x), gr = rows_of(d_y), w = weight.defined() ? weight.contiguous() : weight;
    const at::Tensor mn = mean.contiguous(), rs = rstd.contiguous();
    at::Tensor dx, dw, db;
    if (want_x) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (want_w) dw = at::empty({c}, x.options().dtype(grad_type));
    if (want_b) db = at::empty({c}, x.options().dtype(grad_type));
    hstu_layer_norm_bwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.dtype = type_code(x.scalar_type(), LN, "x");
    p.param_dtype = type_code(param_type, LN, "weight");
    p.grad_dtype = type_code(grad_type, LN, "weight");
    p.cols = (int32_t)c;
    p.rows = rows;
    p.x_stride = rows > 1 ? xr.stride(0) : c;
    p.dy_stride = rows > 1 ? gr.stride(0) : c;
    p.d_y = gr.const_data_ptr();
    p.x = xr.const_data_ptr();
    p.weight = w.defined() ? w.const_data_ptr() : nullptr;
    p.mean = (const float*)mn.const_data_ptr();
    p.rstd = (const float*)rs.const_data_ptr();
    p.d_x = want_x ? dx.data_ptr() : nullptr;
    p.d_weight = want_w ? dw.data_ptr() : nullptr;
    p.d_bias = want_b ? db.data_ptr() : nullptr;
    uint64_t bytes = 0;
    int rc = hstu_hip_layer_norm_backward_get_workspace_size(&p, &bytes);
    TORCH_CHECK(rc == HSTU_OK, LN, ": ", hstu_hip_last_error());
    const at::Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    rc = hstu_hip_layer_norm_backward(&p, bytes ? ws.data_ptr() : nullptr, bytes, launch.stream());
    TORCH_CHECK(rc == HSTU_OK, LN, ": ", hstu_hip_last_error());
    return {dx, dw, db};
}

class LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
public:
    // parameters that are not there take no part in the graph: the edges of the others move up
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& weight_,
                              const c10::optional<at::Tensor>& bias_, double eps) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const at::Tensor weight = value(weight_), bias = value(bias_);
        auto outs = ln_forward(x, weight, bias, eps, true);
        ctx->saved_data["has_weight"] = weight.defined();
        ctx->saved_data["has_bias"] = bias.defined();
        ctx->save_for_backward({x, weight, outs[1], outs[2]});
        ctx->saved_data["param_type"] = (int64_t)ln_param_type(x, weight, bias);
        return outs[0];
    }
    static torch::autograd::tensor_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::tensor_list grads) {
        no_double_backward(LN, grads[0]);
        const auto s = ctx->get_saved_variables();
        const auto pt = (at::ScalarType)ctx->saved_data["param_type"].toInt();
        const bool hw = ctx->saved_data["has_weight"].toBool(), hb = ctx->saved_data["has_bias"].toBool();
        auto g = ln_backward(grads[0], s[0], s[1], s[2], s[3], pt, pt, ctx->needs_input_grad(0), hw && ctx->needs_input_grad(1),
                             hb && ctx->needs_input_grad(hw ? 2 : 1));
        return {g[0], g[1], g[2], at::Tensor()};
    }
};

static bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

at::Tensor layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias, double eps) {
    return ln_forward(x, value(weight), value(bias), eps, false)[0];
}
at::Tensor layer_norm_autograd(const at::Tensor& x, const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias, double eps) {
    const at::Tensor w = value(weight), b = value(bias);
    no_tangents(LN, {&x, &w, &b});
    if (!wants_grad({&x, &w, &b})) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return ln_forward(x, w, b, eps, false)[0];
    }
    return LayerNormFunction::apply(x, weight, bias, eps);
}
std::vector<at::Tensor> layer_norm_forward(const at::Tensor& x, const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias, double eps) {
    return ln_forward(x, value(weight), value(bias), eps, true);
}
std::vector<at::Tensor> layer_norm_backward(const at::Tensor& d_out, const at::Tensor& x, const c10::optional<at::Tensor>& weight, const at::Tensor& mean,
                                            const at::Tensor& rstd) {
    const at::Tensor w = value(weight);
    ln_check(x, w, at::Tensor(), 1.0);
    no_tangents(LN, {&d_out, &x, &w, &mean, &rstd});
    TORCH_CHECK(d_out.sizes() == x.sizes() && d_out.scalar_type() == x.scalar_type(), LN, ": d_out must have the shape and dtype of x");
    const int64_t rows = row_count(x);
    for (const at::Tensor* t : {&mean, &rstd})
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->numel() == rows, LN, ": mean and rstd must be float32 with one value for each of the ", rows, " rows");
    return ln_backward(d_out, x, w, mean, rstd, ln_param_type(x, w, at::Tensor()), at::kFloat, true, true, true);
}

// ---- gated_linear ------------------------------------------------------------------------------------------------------
static const char* GL = "mxrec::gated_linear";

static int32_t act_code(c10::string_view name) {
    if (name == "silu") return HSTU_ACT_SILU;
    if (name == "gelu") return HSTU_ACT_GELU;
    TORCH_CHECK(false, GL, ": activation expect 'silu' or 'gelu', but get '", name, "'");
}

static void gl_check(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, bool checkpoint8) {
    TORCH_CHECK(x.defined() && x.dim() >= 1, GL, ": x must have at least 1 dimension");
    type_code(x.scalar_type(), GL, "x");
    const int64_t k = x.size(-1);
    TORCH_CHECK(k >= 1 && k <= HSTU_GATED_MAX_K, GL, ": the last dimension of x must in range:[1,", HSTU_GATED_MAX_K, "], but get ", k);
    TORCH_CHECK(weight.dim() == 2, GL, ": weight must be 2D");
    TORCH_CHECK(weight.size(1) == k, GL, ": weight dim[1] must equal to the last dimension of x (", k, "), but get ", weight.size(1));
    TORCH_CHECK(weight.size(0) >= 2 && weight.size(0) % 2 == 0 && weight.size(0) <= 2 * HSTU_GATED_MAX_F, GL, ": weight dim[0] must be twice a number in range:[1,",
                HSTU_GATED_MAX_F, "] (gate rows, then value rows), but get ", weight.size(0));
    TORCH_CHECK(weight.scalar_type() == x.scalar_type(), GL, ": weight must have the dtype of x, but get ", weight.scalar_type(), " and ", x.scalar_type());
    if (bias.defined()) {
        TORCH_CHECK(bias.dim() == 1 && bias.size(0) == weight.size(0), GL, ": bias must be 1D with the size of weight dim[0] (", weight.size(0), "), but get ", bias.sizes());
        TORCH_CHECK(bias.scalar_type() == x.scalar_type() || bias.scalar_type() == at::kFloat, GL, ": bias dtype expect ", x.scalar_type(), " or float32, but get ",
                    bias.scalar_type());
    }
    TORCH_CHECK(!checkpoint8 || x.scalar_type() != at::kFloat, GL, ": checkpoint8 needs float16 or bfloat16");
}

static std::vector<int64_t> with_last(const at::Tensor& x, int64_t last) {
    auto s = x.sizes().vec();
    s.back() = last;
    return s;
}

// type and shape of a kept z for rows like x, and the shape of what is kept beside it (empty: nothing).  In the upper parts of the 24-bit
// z the gate's and the values' blocks of 32 columns take turns.
struct Kept { at::ScalarType type; std::vector<int64_t> z, aux; };
static Kept kept_like(const at::Tensor& x, int64_t f, bool checkpoint8) {
    const int64_t m = row_count(x), fp = HSTU_GATED_KEPT(f);
    if (checkpoint8) return {at::kFloat8_e4m3fn, {m, 2, fp}, {m, 2, fp / HSTU_PACK8_GROUP}};
    if (x.scalar_type() == at::kFloat) return {at::kFloat, {m, 2, fp}, {}};
    return {at::kBFloat16, {m, fp / 32, 2, 32}, {m, 2, fp}};
}

// {out}, {out, z} (fp32), {out, upper parts of z, lower parts} (16-bit types: z in 24 bits) or {out, codes, exponents}
static std::vector<at::Tensor> gl_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, int32_t act, int32_t keep) {
    gl_check(x, weight, bias, keep == HSTU_KEEP_8BIT);
    no_tangents(GL, {&x, &weight, &bias});
    check_devices(GL, {&x, &weight, &bias});
    Launch launch(x);
    const at::Tensor xr = rows_of(x), w = weight.contiguous(), b = bias.defined() ? bias.contiguous() : bias;
    const int64_t m = row_count(x), f = weight.size(0) / 2;
    std::vector<at::Tensor> outs{at::empty(with_last(x, f), x.options().memory_format(at::MemoryFormat::Contiguous))};
    if (keep != HSTU_KEEP_NONE) {
        const Kept k = kept_like(x, f, keep == HSTU_KEEP_8BIT);
        outs.push_back(at::empty(k.z, x.options().dtype(k.type)));
        if (!k.aux.empty()) outs.push_back(at::empty(k.aux, x.options().dtype(at::kByte)));
    }
    hstu_gated_params p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.dtype = type_code(x.scalar_type(), GL, "x");
    p.bias_dtype = b.defined() ? type_code(b.scalar_type(), GL, "bias") : p.dtype;
    p.act = act;
    p.keep = keep;
    p.k = (int32_t)x.size(-1);
    p.f = (int32_t)f;
    p.m = m;
    p.x_stride = m > 1 ? xr.stride(0) : p.k;
    p.x = xr.const_data_ptr();
    p.weight = w.const_data_ptr();
    p.bias = b.defined() ? b.const_data_ptr() : nullptr;
    p.out = outs[0].data_ptr();
    p.z = keep != HSTU_KEEP_NONE ? outs[1].data_ptr() : nullptr;
    p.z_aux = outs.size() > 2 ? outs[2].data_ptr<uint8_t>() : nullptr;
    uint64_t bytes = 0;
    int rc = hstu_hip_gated_linear_get_workspace_size(&p, &bytes);
    TORCH_CHECK(rc == HSTU_OK, GL, ": ", hstu_hip_last_error());
    at::Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    rc = hstu_hip_gated_linear(&p, bytes ? ws.data_ptr() : nullptr, bytes, launch.stream());
    TORCH_CHECK(rc == HSTU_OK, GL, ": ", hstu_hip_last_error());
    return outs;
}

// {d_x, d_weight, d_bias}, undefined where not wanted
static std::vector<at::Tensor> gl_backward(const at::Tensor& d_out, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& z, const at::Tensor& aux,
                                           int32_t act, at::ScalarType bias_type, bool want_x, bool want_w, bool want_b) {
    check_devices(GL, {&x, &weight, &d_out, &z, &aux});
    Launch launch(x);
    const at::Tensor xr = rows_of(x), gr = rows_of(d_out), w = weight.contiguous(), zc = z.contiguous(), ac = aux.defined() ? aux.contiguous() : aux;
    const int64_t m = row_count(x), f = weight.size(0) / 2;
    at::Tensor dx, dw, db;
    if (want_x) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (want_w) dw = at::empty(weight.sizes(), weight.options().memory_format(at::MemoryFormat::Contiguous));
    if (want_b) db = at::empty({2 * f}, x.options().dtype(bias_type));
    hstu_gated_bwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.dtype = type_code(x.scalar_type(), GL, "x");
    p.grad_bias_dtype = type_code(bias_type, GL, "bias");
    p.act = act;
    p.keep = z.scalar_type() == at::kFloat8_e4m3fn ? HSTU_KEEP_8BIT : HSTU_KEEP_FULL;
    p.k = (int32_t)x.size(-1);
    p.f = (int32_t)f;
    p.m = m;
    p.x_stride = m > 1 ? xr.stride(0) : p.k;
    p.dout_stride = m > 1 ? gr.stride(0) : f;
    p.d_out = gr.const_data_ptr();
    p.x = xr.const_data_ptr();
    p.weight = w.const_data_ptr();
    p.z = zc.const_data_ptr();
    p.z_aux = ac.defined() ? (const uint8_t*)ac.const_data_ptr() : nullptr;
    p.d_x = want_x ? dx.data_ptr() : nullptr;
    p.d_weight = want_w ? dw.data_ptr() : nullptr;
    p.d_bias = want_b ? db.data_ptr() : nullptr;
    uint64_t bytes = 0;
    int rc = hstu_hip_gated_linear_backward_get_workspace_size(&p, &bytes);
    TORCH_CHECK(rc == HSTU_OK, GL, ": ", hstu_hip_last_error());
    at::Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    rc = hstu_hip_gated_linear_backward(&p, bytes ? ws.data_ptr() : nullptr, bytes, launch.stream());
    TORCH_CHECK(rc == HSTU_OK, GL, ": ", hstu_hip_last_error());
    return {dx, dw, db};
}

class GatedLinearFunction : public torch::autograd::Function<GatedLinearFunction> {
public:
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& bias_,
                              int64_t act, bool checkpoint8) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const at::Tensor bias = value(bias_);
        auto outs = gl_forward(x, weight, bias, (int32_t)act, checkpoint8 ? HSTU_KEEP_8BIT : HSTU_KEEP_FULL);
        ctx->save_for_backward({x, weight, outs[1], outs.size() > 2 ? outs[2] : at::Tensor()});
        ctx->saved_data["act"] = act;
        ctx->saved_data["has_bias"] = bias.defined();
        ctx->saved_data["bias_type"] = (int64_t)(bias.defined() ? bias.scalar_type() : x.scalar_type());
        return outs[0];
    }
    static torch::autograd::tensor_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::tensor_list grads) {
        no_double_backward(GL, grads[0]);
        const auto s = ctx->get_saved_variables();
        auto g = gl_backward(grads[0], s[0], s[1], s[2], s[3], (int32_t)ctx->saved_data["act"].toInt(), (at::ScalarType)ctx->saved_data["bias_type"].toInt(),
                             ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(2));
        return {g[0], g[1], g[2], at::Tensor(), at::Tensor()};
    }
};

at::Tensor gated_linear(const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& bias, c10::string_view activation, bool checkpoint8) {
    gl_check(x, weight, value(bias), checkpoint8);
    return gl_forward(x, weight, value(bias), act_code(activation), HSTU_KEEP_NONE)[0];
}
at::Tensor gated_linear_autograd(const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& bias, c10::string_view activation,
                                 bool checkpoint8) {
    const at::Tensor b = value(bias);
    no_tangents(GL, {&x, &weight, &b});
    if (!wants_grad({&x, &weight, &b})) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return gated_linear(x, weight, bias, activation, checkpoint8);
    }
    return GatedLinearFunction::apply(x, weight, bias, (int64_t)act_code(activation), checkpoint8);
}
std::vector<at::Tensor> gated_linear_forward(const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& bias, c10::string_view activation,
                                             bool checkpoint8) {
    return gl_forward(x, weight, value(bias), act_code(activation), checkpoint8 ? HSTU_KEEP_8BIT : HSTU_KEEP_FULL);
}
std::vector<at::Tensor> gated_linear_backward(const at::Tensor& d_out, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& z,
                                              const c10::optional<at::Tensor>& z_aux, c10::string_view activation) {
    const at::Tensor aux = value(z_aux);
    const bool c8 = z.scalar_type() == at::kFloat8_e4m3fn;
    gl_check(x, weight, at::Tensor(), c8);
    no_tangents(GL, {&d_out, &x, &weight, &z});
    const int64_t f = weight.size(0) / 2;
    const Kept k = kept_like(x, f, c8);
    TORCH_CHECK(d_out.scalar_type() == x.scalar_type() && d_out.sizes().vec() == with_last(x, f), GL, ": d_out must have the dtype of x and the shape of out");
    TORCH_CHECK(z.scalar_type() == k.type && z.sizes().vec() == k.z, GL, ": z must be what gated_linear_forward kept: ", k.type, " ", at::IntArrayRef(k.z));
    const bool two = !k.aux.empty();
    TORCH_CHECK(!two || (aux.defined() && aux.scalar_type() == at::kByte && aux.sizes().vec() == k.aux), GL,
                ": z_aux must be what gated_linear_forward kept beside z: uint8 ", at::IntArrayRef(k.aux));
    return gl_backward(d_out, x, weight, z, two ? aux : at::Tensor(), act_code(activation), at::kFloat, true, true, true);
}

// ---- 8-bit activations ---------------------------------------------------------------------------------------------------
static hstu_pack8_params pack8_params(const char* op, at::ScalarType type, int64_t rows, int64_t cols) {
    TORCH_CHECK(cols >= 1 && cols <= HSTU_PACK8_MAX_COLS, op, ": the last dimension must in range:[1,", HSTU_PACK8_MAX_COLS, "], but get ", cols);
    hstu_pack8_params p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.dtype = type_code(type, op, "activation");
    p.rows = rows;
    p.cols = (int32_t)cols;
    p.x_stride = cols;
    return p;
}

std::vector<at::Tensor> activation_pack8(const at::Tensor& x) {
    const char* op = "mxrec::activation_pack8";
    TORCH_CHECK(x.defined() && x.dim() >= 1, op, ": x must have at least 1 dimension");
    const int64_t rows = row_count(x), cols = x.size(-1);
    hstu_pack8_params p = pack8_params(op, x.scalar_type(), rows, cols);
    no_tangents(op, {&x});
    check_devices(op, {&x});
    Launch launch(x);
    const at::Tensor xr = rows_of(x);
    at::Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn).memory_format(at::MemoryFormat::Contiguous));
    at::Tensor exps = at::empty(with_last(x, (cols + HSTU_PACK8_GROUP - 1) / HSTU_PACK8_GROUP), x.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
    if (rows > 1) p.x_stride = xr.stride(0);
    p.x = const_cast<void*>(xr.const_data_ptr());
    p.codes = (uint8_t*)codes.data_ptr();
    p.exponents = exps.data_ptr<uint8_t>();
    const int rc = hstu_hip_activation_pack8(&p, launch.stream());
    TORCH_CHECK(rc == HSTU_OK, op, ": ", hstu_hip_last_error());
    return {codes, exps};
}

at::Tensor activation_unpack8(const at::Tensor& codes, const at::Tensor& exponents, at::ScalarType dtype) {
    const char* op = "mxrec::activation_unpack8";
    TORCH_CHECK(codes.defined() && codes.dim() >= 1 && codes.scalar_type() == at::kFloat8_e4m3fn, op, ": codes must be float8_e4m3fn with at least 1 dimension");
    const int64_t rows = row_count(codes), cols = codes.size(-1);
    hstu_pack8_params p = pack8_params(op, dtype, rows, cols);
    TORCH_CHECK(exponents.scalar_type() == at::kByte && exponents.sizes().vec() == with_last(codes, (cols + HSTU_PACK8_GROUP - 1) / HSTU_PACK8_GROUP), op,
                ": exponents must be uint8 with the shape of codes and ceil(", cols, " / 32) values along the last dimension, but get ", exponents.scalar_type(), " ",
                exponents.sizes());
    no_tangents(op, {&codes});
    check_devices(op, {&codes, &exponents});
    Launch launch(codes);
    const at::Tensor cc = codes.contiguous(), ec = exponents.contiguous();
    at::Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
    p.x = out.data_ptr();
    p.codes = (uint8_t*)const_cast<void*>(cc.const_data_ptr());
    p.exponents = (uint8_t*)const_cast<void*>(ec.const_data_ptr());
    const int rc = hstu_hip_activation_unpack8(&p, launch.stream());
    TORCH_CHECK(rc == HSTU_OK, op, ": ", hstu_hip_last_error());
    return out;
}

// The plain ops have no backward: under autograd, with an input that asks for gradients, they refuse instead of losing them.
template <typename Fn, Fn fn> struct NoGrad;
template <typename R, typename... Args, R (*fn)(Args...)> struct NoGrad<R (*)(Args...), fn> {
    static bool asks(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
    static bool asks(const c10::optional<at::Tensor>& t) { return t.has_value() && asks(*t); }
    template <typename T> static bool asks(const T&) { return false; }
    static R call(Args... args) {
        TORCH_CHECK(!at::GradMode::is_enabled() || !(asks(args) || ...),
                    "mxrec: this op has no backward: call it under torch.no_grad(), on detached tensors, or use layer_norm / gated_linear");
        at::AutoDispatchBelowADInplaceOrView guard;
        return fn(args...);
    }
};
#define FFN_NO_GRAD(f) TORCH_FN((NoGrad<decltype(&f), &f>::call))

TORCH_LIBRARY_FRAGMENT(mxrec, m) {
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps=1e-05) -> Tensor");
    m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps=1e-05) -> Tensor[]");
    m.def("layer_norm_backward(Tensor d_out, Tensor x, Tensor? weight, Tensor mean, Tensor rstd) -> Tensor[]");
    m.def("gated_linear(Tensor x, Tensor weight, Tensor? bias=None, str activation='silu', bool checkpoint8=False) -> Tensor");
    m.def("gated_linear_forward(Tensor x, Tensor weight, Tensor? bias=None, str activation='silu', bool checkpoint8=False) -> Tensor[]");
    m.def("gated_linear_backward(Tensor d_out, Tensor x, Tensor weight, Tensor z, Tensor? z_aux=None, str activation='silu') -> Tensor[]");
    m.def("activation_pack8(Tensor x) -> Tensor[]");
    m.def("activation_unpack8(Tensor codes, Tensor exponents, ScalarType dtype) -> Tensor");
}

#define FFN_IMPLS(m)                                                \
    m.impl("layer_norm", TORCH_FN(layer_norm));                     \
    m.impl("layer_norm_forward", TORCH_FN(layer_norm_forward));     \
    m.impl("layer_norm_backward", TORCH_FN(layer_norm_backward));   \
    m.impl("gated_linear", TORCH_FN(gated_linear));                 \
    m.impl("gated_linear_forward", TORCH_FN(gated_linear_forward)); \
    m.impl("gated_linear_backward", TORCH_FN(gated_linear_backward)); \
    m.impl("activation_pack8", TORCH_FN(activation_pack8));         \
    m.impl("activation_unpack8", TORCH_FN(activation_unpack8));

// ROCm tensors dispatch on the CUDA key; the CPU key runs the same checks and then reports that there is no CPU implementation
TORCH_LIBRARY_IMPL(mxrec, CUDA, m) { FFN_IMPLS(m) }
TORCH_LIBRARY_IMPL(mxrec, CPU, m) { FFN_IMPLS(m) }
TORCH_LIBRARY_IMPL(mxrec, AutogradCUDA, m) {
    m.impl("layer_norm", TORCH_FN(layer_norm_autograd));
    m.impl("gated_linear", TORCH_FN(gated_linear_autograd));
    m.impl("layer_norm_forward", FFN_NO_GRAD(layer_norm_forward));
    m.impl("layer_norm_backward", FFN_NO_GRAD(layer_norm_backward));
    m.impl("gated_linear_forward", FFN_NO_GRAD(gated_linear_forward));
    m.impl("gated_linear_backward", FFN_NO_GRAD(gated_linear_backward));
    m.impl("activation_pack8", FFN_NO_GRAD(activation_pack8));
    m.impl("activation_unpack8", FFN_NO_GRAD(activation_unpack8));
}

}  // namespace mxrec_ffn
