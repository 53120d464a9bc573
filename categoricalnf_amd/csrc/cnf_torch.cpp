// Host side of the training step's operators: argument checks, outputs, workspaces, autograd nodes and the packing of tensor lists,
// for calls whose kernels take less time than a Python autograd node or a Python loop over the tensors costs.  No arithmetic here:
// every function ends in the C entry points of libcnf_hip.so (include/cnf_hip.h), whose addresses Python hands over once (`bind`), so
// that there is one loaded library whichever build it is.
//
// Measured beside an MI355X: layer norm step (forward + torch.autograd.grad) 123 us as a Python autograd Function, whose
// backward waits for the interpreter lock on the engine's thread; torch's own 35 us.
#include <algorithm>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/cnf_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&cnf_last_error) last_error;
    decltype(&cnf_layer_norm) layer_norm;
    decltype(&cnf_layer_norm_bwd) layer_norm_bwd;
    decltype(&cnf_layer_norm_bwd_workspace_floats) layer_norm_bwd_workspace_floats;
    decltype(&cnf_linear_ce) linear_ce;
    decltype(&cnf_linear_ce_bwd) linear_ce_bwd;
    decltype(&cnf_linear_ce_workspace_bytes) linear_ce_workspace_bytes;
    decltype(&cnf_adamw_step) adamw_step;
} api;
PyObject* hip_only_error = nullptr;

void bind(const std::unordered_map<std::string, uintptr_t>& at, py::object hip_only) {
    auto take = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name)); };
    take(api.last_error, "cnf_last_error");
    take(api.layer_norm, "cnf_layer_norm");
    take(api.layer_norm_bwd, "cnf_layer_norm_bwd");
    take(api.layer_norm_bwd_workspace_floats, "cnf_layer_norm_bwd_workspace_floats");
    take(api.linear_ce, "cnf_linear_ce");
    take(api.linear_ce_bwd, "cnf_linear_ce_bwd");
    take(api.linear_ce_workspace_bytes, "cnf_linear_ce_workspace_bytes");
    take(api.adamw_step, "cnf_adamw_step");
    hip_only_error = hip_only.release().ptr();
}

// ---- checks ----------------------------------------------------------------------------------------------------------------------

// Outputs are allocated by operators and filled through their pointers: a recording of the call would hold the empty tensors alone
void refuse_transforms(const char* name) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                name, " is a HIP kernel, which torch.jit.trace and make_fx cannot record");
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode), name, " is a HIP kernel, which torch.func cannot transform");
}

void need_gpu(const Tensor& t, const char* name) {
    if (t.is_cuda()) return;
    PyErr_Format(hip_only_error, "categoricalnf_amd kernels run on MI355X only: expected %s as a CUDA(HIP) tensor, got %s. There is no CPU fallback.",
                 name, t.device().str().c_str());
    throw py::error_already_set();
}

// a tangent (forward-mode derivative) would be dropped: the kernels have none
void refuse_tangents(std::initializer_list<const Tensor*> ts, const char* name) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, " is a HIP kernel without a forward-mode derivative");
}

int dtype_code(const Tensor& t, const char* name) {
    need_gpu(t, name);
    switch (t.scalar_type()) {
        case at::kFloat: return CNF_DTYPE_F32;
        case at::kBFloat16: return CNF_DTYPE_BF16;
        case at::kHalf: return CNF_DTYPE_F16;
        default: TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

// an optional parameter vector of n elements, dense
Tensor vector_of(const Tensor& t, int64_t n, const char* name, const at::Device& device) {
    if (!t.defined()) return t;
    dtype_code(t, name);
    TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", the input on ", device);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " must have shape (", n, ",), got ", t.sizes());
    return t.contiguous();
}

// [..., C] as [rows, C] with unit column stride and one row stride: a view where the strides allow it, else a copy
Tensor rows_of(const Tensor& t) {
    Tensor m = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}

// an empty tensor has a null data pointer, which the entry points refuse; they return before touching memory then
void* ptr(const Tensor& t) { return !t.defined() ? nullptr : (t.numel() ? t.data_ptr() : reinterpret_cast<void*>(16)); }

cnf_stream_t stream_of(const at::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

void check(int status, const char* name) { TORCH_CHECK(status == CNF_OK, name, " failed with status ", status, ": ", api.last_error()); }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// gradients of a backward that has none itself: differentiating them again raises
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function whose backward is a HIP kernel without a derivative", (int64_t)grads.size());
    return (*error)(std::move(grads));
}

Tensor opt(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// ---- layer norm --------------------------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> layer_norm_raw(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool want_stats) {
    refuse_transforms("layer_norm");
    refuse_tangents({&x, &weight, &bias}, "layer_norm");
    const int code = dtype_code(x, "x");
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "layer_norm needs a last axis of at least one element, got shape ", x.sizes());
    TORCH_CHECK_VALUE(x.size(-1) <= 1 << 30, "layer_norm: ", x.size(-1), " columns");
    const int64_t C = x.size(-1);
    const Tensor w = vector_of(weight, C, "weight", x.device()), b = vector_of(bias, C, "bias", x.device());
    TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight is ", w.defined() ? w.scalar_type() : at::kFloat,
                     ", bias ", b.defined() ? b.scalar_type() : at::kFloat);
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = rows_of(x);
    const int64_t R = x2.size(0);
    Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous), mean, rstd;
    if (want_stats) {
        mean = at::empty({2, R}, x.options().dtype(at::kFloat));
        rstd = mean.select(0, 1);
        mean = mean.select(0, 0);
    }
    const int wcode = w.defined() ? dtype_code(w, "weight") : (b.defined() ? dtype_code(b, "bias") : CNF_DTYPE_F32);
    check(api.layer_norm(ptr(x2), x2.stride(0), ptr(w), ptr(b), ptr(y), static_cast<float*>(ptr(mean)), static_cast<float*>(ptr(rstd)), R, (int)C,
                         (float)eps, code, wcode, stream_of(x.device())),
          "cnf_layer_norm");
    return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd_raw(const Tensor& x, const Tensor& dy, const Tensor& weight, const Tensor& mean, const Tensor& rstd,
                                                      at::ScalarType pdtype, bool want_weight, bool want_bias) {
    refuse_transforms("layer_norm_bwd");
    refuse_tangents({&x, &dy, &weight}, "layer_norm_bwd");
    const int code = dtype_code(x, "x");
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0 && x.size(-1) <= 1 << 30, "layer_norm_bwd needs a last axis of 1 to 2^30 elements, got shape ",
                      x.sizes());
    const int64_t C = x.size(-1);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
                      "the gradient must have the input's shape and type, got ", dy.sizes(), " ", dy.scalar_type(), " for ", x.sizes(), " ",
                      x.scalar_type());
    const Tensor w = vector_of(weight, C, "weight", x.device());
    TORCH_CHECK_TYPE(!w.defined() || w.scalar_type() == pdtype, "parameter gradients have the weight's type");
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = rows_of(x), g2 = rows_of(dy);
    const int64_t R = x2.size(0);
    TORCH_CHECK_VALUE(mean.numel() == R && rstd.numel() == R && mean.is_contiguous() && rstd.is_contiguous() && mean.scalar_type() == at::kFloat &&
                          rstd.scalar_type() == at::kFloat && mean.device() == x.device() && rstd.device() == x.device(),
                      "mean and rstd are the forward's: [", R, "] float32");
    Tensor dx = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous), dw, db, ws;
    const auto popt = x.options().dtype(pdtype);
    if (want_weight) dw = at::empty({C}, popt);
    if (want_bias) db = at::empty({C}, popt);
    int64_t n = 0;
    if (want_weight || want_bias) {
        n = api.layer_norm_bwd_workspace_floats(R, (int)C);
        ws = at::empty({n}, x.options().dtype(at::kFloat));
    }
    const int pcode = pdtype == at::kFloat ? CNF_DTYPE_F32 : (pdtype == at::kBFloat16 ? CNF_DTYPE_BF16 : CNF_DTYPE_F16);
    check(api.layer_norm_bwd(ptr(x2), x2.stride(0), ptr(g2), g2.stride(0), ptr(w), static_cast<const float*>(ptr(mean)),
                             static_cast<const float*>(ptr(rstd)), ptr(dx), ptr(dw), ptr(db), static_cast<float*>(ptr(ws)), n, R, (int)C, code, pcode,
                             stream_of(x.device())),
          "cnf_layer_norm_bwd");
    return {dx, dw, db};
}

// the gradients as operators that autograd knows, for a backward that is differentiated itself, batched or given a tangent
variable_list layer_norm_bwd_composed(const Tensor& x, const Tensor& dy, const Tensor& weight, at::ScalarType pdtype, double eps, bool want_weight,
                                      bool want_bias) {
    const Tensor xf = x.to(at::kFloat), g = dy.to(at::kFloat), gw = weight.defined() ? g * weight.to(at::kFloat) : g;
    const Tensor centred = xf - xf.mean(-1, true), rstd = (centred.square().mean(-1, true) + eps).rsqrt(), xhat = centred * rstd;
    const Tensor dx = rstd * (gw - gw.mean(-1, true) - xhat * (gw * xhat).mean(-1, true));
    auto columns = [&](const Tensor& t) { return t.reshape({-1, x.size(-1)}).sum(0).to(pdtype); };
    return {dx.to(x.scalar_type()), want_weight ? columns(g * xhat) : Tensor(), want_bias ? columns(g) : Tensor(), Tensor(), Tensor()};
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    // an absent parameter is no input of the node: the others' places in needs_input_grad move up
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w, const std::optional<Tensor>& b, double eps, bool twice) {
        const Tensor weight = opt(w), bias = opt(b);
        auto [y, mean, rstd] = layer_norm_raw(x, weight, bias, eps, true);
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["twice"] = twice;
        ctx->save_for_backward({x, weight, mean, rstd});
        ctx->saved_data["dtype"] = (int64_t)(weight.defined() ? weight.scalar_type() : (bias.defined() ? bias.scalar_type() : x.scalar_type()));
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const auto pdtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
        const bool want_weight = s[1].defined() && ctx->needs_input_grad(1);
        const bool want_bias = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(s[1].defined() ? 2 : 1);
        // (batched gradients are wrappers without memory of their own)
        if (ctx->saved_data["twice"].toBool() && (at::GradMode::is_enabled() || !g[0].has_storage() || g[0]._fw_grad(0).defined()))
            return layer_norm_bwd_composed(s[0], g[0], s[1], pdtype, ctx->saved_data["eps"].toDouble(), want_weight, want_bias);
        auto [dx, dw, db] = layer_norm_bwd_raw(s[0], g[0], s[1], s[2], s[3], pdtype, want_weight, want_bias);
        return once({dx, dw, db, Tensor(), Tensor()});
    }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps, bool twice) {
    const Tensor w = opt(weight), b = opt(bias);
    refuse_transforms("layer_norm");
    refuse_tangents({&x, &w, &b}, "layer_norm");
    if (wants_grad({&x, &w, &b})) return LayerNormNode::apply(x, weight, bias, eps, twice);
    return std::get<0>(layer_norm_raw(x, w, b, eps, false));
}

// ---- linear cross entropy -----------------------------------------------------------------------------------------------------------

struct CeOperands {
    Tensor x, w, b, t;
    int64_t R, V, H;
    int code, bcode;
};

CeOperands ce_operands(const Tensor& x, const Tensor& weight, const Tensor& target, const Tensor& bias) {
    CeOperands o;
    o.code = dtype_code(x, "x");
    need_gpu(weight, "weight");
    need_gpu(target, "target");
    TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "x is ", x.scalar_type(), ", weight ", weight.scalar_type());
    TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() >= 1 && weight.size(1) == x.size(-1) && weight.numel() > 0,
                      "weight must be [V, H] with the H of x, both at least 1: got ", weight.sizes(), " for x ", x.sizes());
    TORCH_CHECK_TYPE(target.scalar_type() == at::kLong || target.scalar_type() == at::kInt, "target must hold integers (int64 or int32), got ",
                     target.scalar_type());
    TORCH_CHECK_VALUE(target.sizes() == x.sizes().slice(0, x.dim() - 1), "target must have the shape of x without its last axis: got ", target.sizes(),
                      " for ", x.sizes());
    TORCH_CHECK_VALUE(weight.device() == x.device() && target.device() == x.device(), "weight is on ", weight.device(), ", target on ", target.device(),
                      ", x on ", x.device());
    o.V = weight.size(0);
    o.H = weight.size(1);
    o.R = target.numel();
    TORCH_CHECK_VALUE(o.V <= 1 << 30 && o.H <= 1 << 21 && o.R <= 0x7fffff00, "linear_cross_entropy: sizes ", o.R, " x ", o.V, " x ", o.H);
    o.b = vector_of(bias, o.V, "bias", x.device());
    o.bcode = o.b.defined() ? dtype_code(o.b, "bias") : CNF_DTYPE_F32;
    TORCH_CHECK_TYPE(o.bcode == o.code || o.bcode == CNF_DTYPE_F32, "bias is float32 or of the weight's type, got ", o.b.scalar_type());
    o.x = rows_of(x);
    o.w = rows_of(weight);
    o.t = target.reshape({-1}).to(at::kLong).contiguous();
    return o;
}

// loss, row statistics [2][R] (maximum, sum), reduced [3] or none, exponents [2]
std::tuple<Tensor, Tensor, Tensor, Tensor> linear_ce_raw(const Tensor& x, const Tensor& weight, const Tensor& target, const Tensor& bias,
                                                         int64_t ignore_index, bool want_reduced, const Tensor& flags) {
    refuse_transforms("linear_cross_entropy");
    refuse_tangents({&x, &weight, &bias}, "linear_cross_entropy");
    const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::optional<at::Device>(x.device()) : std::nullopt);
    const CeOperands o = ce_operands(x, weight, target, bias);
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor loss = at::empty(target.sizes(), f32), stats = at::empty({2, o.R}, f32), reduced, exps = at::empty({2}, f32.dtype(at::kInt));
    if (want_reduced) reduced = at::empty({3}, f32);
    const int64_t n = api.linear_ce_workspace_bytes(o.R, (int)o.V, (int)o.H, o.code, 0);
    const Tensor ws = at::empty({n}, f32.dtype(at::kByte));
    float* m = static_cast<float*>(ptr(stats));
    check(api.linear_ce(ptr(o.x), o.x.stride(0), ptr(o.w), o.w.stride(0), ptr(o.b), static_cast<const int64_t*>(ptr(o.t)), ignore_index,
                        static_cast<float*>(ptr(loss)), m, m + o.R, static_cast<float*>(ptr(reduced)), static_cast<int*>(ptr(exps)), ptr(ws), n, o.R,
                        (int)o.V, (int)o.H, o.code, o.bcode, static_cast<int*>(ptr(flags)), stream_of(x.device())),
          "cnf_linear_ce");
    return {loss, stats, reduced, exps};
}

std::tuple<Tensor, Tensor, Tensor> linear_ce_bwd_raw(const Tensor& x, const Tensor& weight, const Tensor& target, const Tensor& bias,
                                                     const Tensor& stats, const Tensor& exps, const Tensor& g, const Tensor& count,
                                                     int64_t ignore_index, bool want_x, bool want_w, bool want_b) {
    refuse_transforms("linear_cross_entropy_bwd");
    refuse_tangents({&x, &weight, &bias, &g}, "linear_cross_entropy_bwd");
    const c10::DeviceGuard guard(x.device());
    const CeOperands o = ce_operands(x, weight, target, bias);
    want_b = want_b && o.b.defined();
    Tensor dx, dw, db;
    if (want_x) dx = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
    if (want_w || want_b) dw = at::empty({o.V, o.H}, x.options());
    if (want_b) db = at::empty({o.V}, o.b.options());
    if (o.R == 0) {
        if (dw.defined()) dw.zero_();
        if (db.defined()) db.zero_();
        return {dx, want_w ? dw : Tensor(), db};
    }
    if (!dx.defined() && !dw.defined()) return {dx, dw, db};
    const Tensor gc = g.reshape({-1}).contiguous();
    TORCH_CHECK_VALUE(gc.scalar_type() == at::kFloat && gc.device() == x.device() && gc.numel() == (count.defined() ? 1 : o.R),
                      "the upstream gradient has ", gc.numel(), " values of ", gc.scalar_type(), " for ", o.R, " rows");
    for (const Tensor* s : {&stats, &count, &exps})
        TORCH_CHECK_VALUE(!s->defined() || (s->device() == x.device() && s->is_contiguous()), "row statistics are the forward's");
    TORCH_CHECK_VALUE(stats.numel() == 2 * o.R && stats.scalar_type() == at::kFloat &&
                          (!count.defined() || (count.scalar_type() == at::kFloat && count.numel() == 1)) &&
                          (!exps.defined() || (exps.numel() == 2 && exps.scalar_type() == at::kInt)),
                      "row statistics are the forward's: [2, ", o.R, "] float32");
    const int64_t n = api.linear_ce_workspace_bytes(o.R, (int)o.V, (int)o.H, o.code, 1);
    const Tensor ws = at::empty({n}, x.options().dtype(at::kByte));
    const float* m = static_cast<const float*>(ptr(stats));
    check(api.linear_ce_bwd(ptr(o.x), o.x.stride(0), ptr(o.w), o.w.stride(0), ptr(o.b), static_cast<const int64_t*>(ptr(o.t)), ignore_index, m,
                            m + o.R, static_cast<const int*>(ptr(exps)), static_cast<const float*>(ptr(gc)), !count.defined(),
                            static_cast<const float*>(ptr(count)), ptr(dx), ptr(dw), ptr(db), ptr(ws), n, o.R, (int)o.V, (int)o.H, o.code, o.bcode,
                            stream_of(x.device())),
          "cnf_linear_ce_bwd");
    return {dx, want_w ? dw : Tensor(), db};
}

enum Reduction { kNone = 0, kMean = 1, kSum = 2 };

// one of the reduced values as a tensor of its own, no view: a caller may change a loss in place while the count is kept for the backward
Tensor value_of(const Tensor& reduced, int64_t k) { return at::empty({0}, reduced.options()).set_(reduced.storage(), k, {}, {}); }

struct LinearCeNode : torch::autograd::Function<LinearCeNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& b, const Tensor& target,
                          int64_t ignore_index, int64_t reduction, const Tensor& flags) {
        const Tensor bias = opt(b);
        auto [loss, stats, reduced, exps] = linear_ce_raw(x, weight, target, bias, ignore_index, reduction != kNone, flags);
        Tensor count;
        if (reduction == kMean) count = value_of(reduced, 2);
        ctx->save_for_backward({x, weight, bias, target, stats, exps, count});
        ctx->saved_data["ignore"] = ignore_index;
        ctx->saved_data["reduction"] = reduction;
        return reduction == kNone ? loss : value_of(reduced, reduction - 1);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const int64_t reduction = ctx->saved_data["reduction"].toInt();
        const Tensor up = reduction == kSum ? g[0].expand({s[3].numel()}) : g[0];
        auto [dx, dw, db] = linear_ce_bwd_raw(s[0], s[1], s[3], s[2], s[4], s[5], up, s[6], ctx->saved_data["ignore"].toInt(),
                                              ctx->needs_input_grad(0), ctx->needs_input_grad(1), s[2].defined() && ctx->needs_input_grad(2));
        return once({dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor linear_ce(const Tensor& x, const Tensor& weight, const Tensor& target, const std::optional<Tensor>& bias, int64_t ignore_index,
                 int64_t reduction, const Tensor& flags) {
    const Tensor b = opt(bias);
    refuse_transforms("linear_cross_entropy");
    refuse_tangents({&x, &weight, &b}, "linear_cross_entropy");
    if (wants_grad({&x, &weight, &b})) return LinearCeNode::apply(x, weight, bias, target, ignore_index, reduction, flags);
    auto [loss, stats, reduced, exps] = linear_ce_raw(x, weight, target, b, ignore_index, reduction != kNone, flags);
    return reduction == kNone ? loss : value_of(reduced, reduction - 1);
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------------------

// the tensors of a Python sequence, by reference: the sequence keeps them alive
struct TensorList {
    py::object fast;
    std::vector<const Tensor*> t;
    TensorList(const py::object& seq, const char* name) {
        PyObject* f = PySequence_Fast(seq.ptr(), "adamw_step takes lists of tensors");
        if (!f) throw py::error_already_set();
        fast = py::reinterpret_steal<py::object>(f);
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(f);
        t.resize(n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PySequence_Fast_GET_ITEM(f, i);
            TORCH_CHECK_TYPE(THPVariable_Check(o), "adamw_step: ", name, " must hold tensors");
            t[i] = &THPVariable_Unpack(o);
        }
    }
};

// no two of the tensors that are written share memory: [list][tensor] addresses, elements and bytes of an element
void check_apart(const std::vector<std::vector<void*>>& at, const std::vector<int64_t>& numel, const std::vector<int64_t>& size, int64_t block) {
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve(at.size() * numel.size());
    for (size_t k = 0; k < at.size(); ++k) {
        if (k == 1) continue;                   // gradients are read only
        for (size_t i = 0; i < numel.size(); ++i)
            if (numel[i]) spans.emplace_back((uintptr_t)at[k][i], (uintptr_t)at[k][i] + (k < 4 ? numel[i] : (numel[i] + block - 1) / block) * size[k]);
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second, "adamw_step: two of the parameters and moments share memory");
}

// a step's number: a host value, or one float32 on the device
std::pair<double, Tensor> scalar(const py::object& v, const char* name, const at::Device& device) {
    if (!THPVariable_Check(v.ptr())) return {v.cast<double>(), Tensor()};
    const Tensor t = THPVariable_Unpack(v.ptr());
    TORCH_CHECK_VALUE(t.device() == device && t.scalar_type() == at::kFloat && t.numel() == 1, name,
                      " as a tensor is one float32 value on the parameters' device, got ", t.scalar_type(), " on ", t.device());
    return {0.0, t};
}

void adamw_step(const py::object& params, const py::object& grads, const py::object& exp_avgs, const py::object& exp_avg_sqs, const py::object& step,
                const py::object& lr, double beta1, double beta2, double eps, double weight_decay, const py::object& exp_avg_scales,
                const py::object& exp_avg_sq_scales, int64_t block) {
    refuse_transforms("adamw_step");
    TORCH_CHECK_VALUE(exp_avg_scales.is_none() == exp_avg_sq_scales.is_none(), "8-bit moments need both lists of scales");
    const bool bits8 = !exp_avg_scales.is_none();
    const char* names[6] = {"params", "grads", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales"};
    const py::object* seqs[6] = {&params, &grads, &exp_avgs, &exp_avg_sqs, &exp_avg_scales, &exp_avg_sq_scales};
    const int lists = bits8 ? 6 : 4;
    std::vector<TensorList> l;
    for (int k = 0; k < lists; ++k) {
        TORCH_CHECK_VALUE(PySequence_Check(seqs[k]->ptr()), "adamw_step: ", names[k], " must be a list of tensors");
        l.emplace_back(*seqs[k], names[k]);
        TORCH_CHECK_VALUE(l[k].t.size() == l[0].t.size(), "adamw_step: ", l[k].t.size(), " ", names[k], " for ", l[0].t.size(), " params");
    }
    const size_t n = l[0].t.size();
    if (n == 0) return;
    const Tensor &p0 = *l[0].t[0], &g0 = *l[1].t[0];
    const int pcode = dtype_code(p0, "params"), gcode = dtype_code(g0, "grads");
    TORCH_CHECK_TYPE(gcode == pcode || gcode == CNF_DTYPE_F32, "gradients are float32 or of the parameters' type, got ", g0.scalar_type(), " for ",
                     p0.scalar_type());
    const at::Device device = p0.device();
    const at::ScalarType types[6] = {p0.scalar_type(), g0.scalar_type(), bits8 ? at::kChar : at::kFloat, bits8 ? at::kByte : at::kFloat, at::kFloat,
                                     at::kFloat};
    std::vector<Tensor> kept;               // dense copies of gradients: alive until the launches are enqueued
    std::vector<std::vector<void*>> at_(lists, std::vector<void*>(n));
    std::vector<int64_t> numel(n);
    const c10::DeviceGuard guard(device);
    for (size_t i = 0; i < n; ++i) {
        numel[i] = l[0].t[i]->numel();
        for (int k = 0; k < lists; ++k) {
            const Tensor* t = l[k].t[i];
            const int64_t want = k < 4 ? numel[i] : (numel[i] + block - 1) / block;
            TORCH_CHECK_VALUE(t->scalar_type() == types[k] && t->numel() == want && t->device() == device && t->layout() == at::kStrided &&
                                  (k == 1 || t->is_contiguous()),
                              "adamw_step: ", names[k], "[", i, "] must be a dense ", types[k], " tensor of ", want, " elements on ", device, ", got ",
                              t->sizes(), " ", t->scalar_type(), " on ", t->device());
            if (k == 1 && !t->is_contiguous()) {
                kept.push_back(t->contiguous());
                t = &kept.back();
                at_[k][i] = t->data_ptr();
                continue;
            }
            at_[k][i] = t->data_ptr();
        }
    }
    check_apart(at_, numel, {p0.element_size(), 0, bits8 ? 1 : 4, bits8 ? 1 : 4, 4, 4}, block);
    TORCH_CHECK_VALUE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw_step: betas outside [0, 1)");
    const auto [step_host, step_dev] = scalar(step, "step", device);
    const auto [lr_host, lr_dev] = scalar(lr, "lr", device);
    TORCH_CHECK_VALUE(step_dev.defined() || step_host >= 1.0, "adamw_step: the first step is step 1, got ", step_host);
    check(api.adamw_step((int)n, at_[0].data(), const_cast<const void* const*>(at_[1].data()), at_[2].data(), at_[3].data(),
                         bits8 ? reinterpret_cast<float* const*>(at_[4].data()) : nullptr,
                         bits8 ? reinterpret_cast<float* const*>(at_[5].data()) : nullptr, numel.data(), pcode, gcode, bits8 ? 8 : 32, lr_host, beta1,
                         beta2, eps, weight_decay, step_host, static_cast<const float*>(ptr(lr_dev)), static_cast<const float*>(ptr(step_dev)),
                         stream_of(device)),
          "cnf_adamw_step");
    // as after any operation in place: a graph that has saved one of these raises in its backward instead of using the new values
    for (int k = 0; k < lists; ++k)
        if (k != 1)
            for (const Tensor* t : l[k].t)
                if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

}  // namespace

PYBIND11_MODULE(_cnf_torch, m) {
    m.def("bind", &bind);
    m.def("refuse_transforms", [](const std::string& name) { refuse_transforms(name.c_str()); });
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_raw", [](const Tensor& x, const std::optional<Tensor>& w, const std::optional<Tensor>& b, double eps, bool stats) {
        return layer_norm_raw(x, opt(w), opt(b), eps, stats);
    });
    m.def("layer_norm_bwd_raw", [](const Tensor& x, const Tensor& dy, const std::optional<Tensor>& w, const Tensor& mean, const Tensor& rstd,
                                   py::object pdtype, bool want_weight, bool want_bias) {
        TORCH_CHECK_TYPE(THPDtype_Check(pdtype.ptr()), "param_dtype must be a torch.dtype");
        const at::ScalarType t = reinterpret_cast<THPDtype*>(pdtype.ptr())->scalar_type;
        TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "parameter gradients are float32, bfloat16 or float16");
        return layer_norm_bwd_raw(x, dy, opt(w), mean, rstd, t, want_weight, want_bias);
    });
    m.def("linear_ce", &linear_ce);
    m.def("linear_ce_raw", [](const Tensor& x, const Tensor& w, const Tensor& t, const std::optional<Tensor>& b, int64_t ignore, bool want_reduced,
                              const Tensor& flags) { return linear_ce_raw(x, w, t, opt(b), ignore, want_reduced, flags); });
    m.def("linear_ce_bwd_raw", [](const Tensor& x, const Tensor& w, const Tensor& t, const std::optional<Tensor>& b, const Tensor& stats,
                                  const std::optional<Tensor>& exps, const Tensor& g, const std::optional<Tensor>& count, int64_t ignore, bool want_x,
                                  bool want_w, bool want_b) {
        return linear_ce_bwd_raw(x, w, t, opt(b), stats, opt(exps), g, opt(count), ignore, want_x, want_w, want_b);
    });
    m.def("adamw_step", &adamw_step);
}
