// bl_torchops.cpp -- _torchops.so: the learner-step operators of libboardlaw_amd.so (bl_logprobs, bl_norm_residual, bl_orthogonalize) as functions
// of torch tensors: argument checks, outputs, workspaces, the current stream of the tensors' device, and the autograd nodes.
//
// Plumbing only (host code, no kernels).  It is C++ because a training step calls these between small kernels: as ctypes calls under a Python
// autograd.Function a forward and backward of one operator took 160 us of host time around 16 us of kernels (log probabilities of
// 32768 rows of 81), most of it in the engine's thread waiting for the interpreter.  Built by boardlaw_amd/build.py with the host compiler
// against torch's headers; like libbl_torchgen.so it is tied to the torch it was built with.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/boardlaw_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

[[noreturn]] void raise(PyObject* type, const std::string& what) {
    PyErr_SetString(type, what.c_str());
    throw py::error_already_set();
}

// ---- argument checks (called with the interpreter's lock) ----
std::string shape_of(at::IntArrayRef s) { std::stringstream o; o << "("; for (size_t i = 0; i < s.size(); i++) o << (i ? ", " : "") << s[i]; o << ")"; return o.str(); }
template <typename... A> std::string say(const A&... a) { std::stringstream o; (o << ... << a); return o.str(); }
template <typename... A> void type_check(bool ok, const A&... a) { if (!ok) raise(PyExc_TypeError, say(a...)); }
template <typename... A> void value_check(bool ok, const A&... a) { if (!ok) raise(PyExc_ValueError, say(a...)); }

int code_of(at::ScalarType t) { return t == at::kFloat ? BL_F32 : t == at::kHalf ? BL_F16 : t == at::kBFloat16 ? BL_BF16 : -1; }

void device_check(const Tensor& first, std::initializer_list<const Maybe*> others) {
    for (const Maybe* o : others)
        if (*o && (*o)->device() != first.device()) raise(PyExc_AssertionError, "Inputs span multiple devices");
    if (!first.is_cuda()) {
        const py::object error = py::module_::import("boardlaw_amd._native").attr("NativeError");
        raise(error.ptr(), say("boardlaw_amd kernels run on an MI355X only: tensors must live on a cuda (HIP) device, got ", first.device(), ". There is no CPU fallback."));
    }
}

// These operators are not torch's, so a tracer (torch.jit.trace, make_fx) would write down their empty outputs and not the call, and a
// forward-mode tangent would be dropped: both without a word, unless refused
bool traced() {
    return at::tracer::impl::is_dispatch_enabled() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
}
void refuse(const std::string& what) { raise(PyExc_NotImplementedError, what); }
void transform_check(const char* name, std::initializer_list<const Maybe*> tensors) {
    if (traced()) refuse(say(name, " cannot be traced: its kernels are not torch's, and the trace would hold their empty outputs"));
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Maybe* t : tensors)
        if (*t && (*t)->_fw_grad(0).defined()) refuse(say(name, " has no forward-mode derivative: got a tensor with a tangent"));
}

void check(int rc) { TORCH_CHECK(rc == BL_OK, "libboardlaw_amd: ", bl_strerror(rc), " (code ", rc, ")"); }

bl_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
long row_stride(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }

// values as they lie in memory: a tensor whose sign is a flag (the imaginary part of a conjugated tensor) is written out
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// (..., width) as (rows, width) with a contiguous last dimension: a view where the layout allows one
Tensor rows_of(const Tensor& t, int64_t width) {
    if (!t.defined()) return t;
    const Tensor p = plain(t), flat = p.dim() == 2 ? p : p.reshape({p.numel() / std::max<int64_t>(width, 1), width});
    return width == 1 || flat.stride(1) == 1 ? flat : flat.contiguous();
}
Tensor solid(const Tensor& t) { return t.defined() ? plain(t).contiguous() : t; }
std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t n) { std::vector<int64_t> s(lead.begin(), lead.end()); s.push_back(n); return s; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
void once() {
    TORCH_CHECK(!at::GradMode::is_enabled(), "this operator is differentiable once: its backward pass does not run under create_graph=True");
    TORCH_CHECK_NOT_IMPLEMENTED(!traced(), "this operator's backward pass cannot be traced");
}

// A saved tensor, or a gradient, as the kernels will read it: a saved-tensor hook may return anything
void kept(const Tensor& t, const Tensor& first, at::IntArrayRef sizes, at::ScalarType type) {
    TORCH_CHECK(!t.defined() || (t.is_cuda() && t.device() == first.device() && t.sizes() == sizes && t.scalar_type() == type),
                "a saved tensor came back from its hook on another device or with another shape or type: ", t.device(), " ", t.scalar_type(), " ", shape_of(t.sizes()),
                " instead of ", first.device(), " ", type, " ", shape_of(sizes));
}

// ---- log probabilities ----
struct LogProbs { Tensor logp, entropy, top, top_logp, stats; };

LogProbs logprobs(const Tensor& raw, const Tensor& actions, const Tensor& valid, int64_t k, bool want_stats) {
    const int64_t R = raw.size(0), A = raw.size(1);
    const auto f32 = raw.options().dtype(at::kFloat).requires_grad(false);
    LogProbs o;
    o.entropy = at::empty({R}, f32);
    if (actions.defined()) o.logp = at::empty({R}, f32);
    if (k) { o.top = at::empty({R, k}, f32.dtype(at::kLong)); o.top_logp = at::empty({R, k}, f32); }
    if (want_stats) o.stats = at::empty({R, 2}, f32);
    if (!R) return o;
    const c10::DeviceGuard guard(raw.device());
    const long size = bl_logprobs_workspace(R, (int)A, (int)k);
    const Tensor work = size ? at::empty({size}, f32.dtype(at::kByte)) : Tensor();
    check(bl_logprobs(ptr(raw), code_of(raw.scalar_type()), raw.stride(0), ptr<uint8_t>(valid), row_stride(valid), ptr<const long long>(actions), R, (int)A,
                      (int)k, ptr<float>(o.logp), ptr<float>(o.entropy), ptr<long long>(o.top), ptr<float>(o.top_logp), ptr<float>(o.stats), ptr(work), stream_of(raw)));
    return o;
}

struct LogProbsNode : torch::autograd::Function<LogProbsNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& raw, const Maybe& actions, const Maybe& valid, int64_t k) {
        const LogProbs o = logprobs(raw, value(actions), value(valid), k, true);
        ctx->save_for_backward({raw, value(actions), value(valid), o.top, o.stats, o.entropy});
        ctx->set_materialize_grads(false);
        ctx->saved_data["k"] = k; ctx->saved_data["A"] = raw.size(1);
        ctx->saved_data["given"] = o.logp.defined();
        if (o.top.defined()) ctx->mark_non_differentiable({o.top});
        variable_list out = {o.entropy};
        if (o.logp.defined()) out.push_back(o.logp);
        if (k) { out.push_back(o.top_logp); out.push_back(o.top); }
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        TORCH_CHECK(s[0].dim() == 2 && code_of(s[0].scalar_type()) >= 0, "a saved tensor came back from its hook with another shape or type");
        const int64_t R = s[0].size(0), A = ctx->saved_data["A"].toInt(), k = ctx->saved_data["k"].toInt();
        kept(s[0], s[4], {R, A}, s[0].scalar_type());
        kept(s[1], s[0], {R}, at::kLong); kept(s[2], s[0], {R, A}, at::kBool); kept(s[3], s[0], {R, k}, at::kLong); kept(s[4], s[0], {R, 2}, at::kFloat); kept(s[5], s[0], {R}, at::kFloat);
        // (a saved-tensor hook may return them with other strides)
        const Tensor raw = rows_of(s[0], A), actions = solid(s[1]), valid = rows_of(s[2], A), top = solid(s[3]), stats = solid(s[4]), entropy = solid(s[5]);
        const bool given = ctx->saved_data["given"].toBool();
        const Tensor d = at::empty({R, A}, raw.options());
        if (R) {
            const Tensor g_entropy = solid(g[0]), g_logp = given ? solid(g[1]) : Tensor(), g_top = k ? solid(g[given ? 2 : 1]) : Tensor();
            kept(g_entropy, raw, {R}, at::kFloat); kept(g_logp, raw, {R}, at::kFloat); kept(g_top, raw, {R, k}, at::kFloat);
            const c10::DeviceGuard guard(raw.device());
            check(bl_logprobs_grad(ptr(raw), code_of(raw.scalar_type()), raw.stride(0), ptr<uint8_t>(valid), row_stride(valid), ptr<const long long>(actions), R, (int)A,
                                   (int)k, ptr<const long long>(top), ptr<float>(stats), ptr<float>(entropy), ptr<float>(g_logp), ptr<float>(g_entropy), ptr<float>(g_top),
                                   ptr(d), stream_of(raw)));
        }
        return {d, Tensor(), Tensor(), Tensor()};
    }
};

py::tuple py_logprobs(const Tensor& raw, const Maybe& actions, const Maybe& valid, int64_t k) {
    type_check(code_of(raw.scalar_type()) >= 0, "raw must be float32, float16 or bfloat16, got ", raw.scalar_type());
    value_check(raw.dim() >= 1 && raw.size(-1) >= 1, "raw must be (..., A) with at least one move, got ", shape_of(raw.sizes()));
    value_check(k >= 0 && k <= BL_TOP_MAX, "k must be in 0 .. ", BL_TOP_MAX, ", got ", k);
    const Maybe raw_ = raw;
    transform_check("logprobs", {&raw_, &actions, &valid});
    device_check(raw, {&actions, &valid});
    const auto lead = raw.sizes().slice(0, raw.dim() - 1);
    const int64_t A = raw.size(-1);
    value_check(A <= BL_LOGPROBS_MAX && raw.numel() / A <= BL_LOGPROBS_ROWS, "up to ", BL_LOGPROBS_ROWS, " rows of up to ", BL_LOGPROBS_MAX, " moves are supported, got ", shape_of(raw.sizes()));
    const Tensor flat = rows_of(raw, A);
    Maybe a, v;
    if (actions) {
        value_check(actions->sizes() == lead, "actions must be ", shape_of(lead), ", got ", shape_of(actions->sizes()));
        type_check(at::isIntegralType(actions->scalar_type(), false), "actions must be whole numbers, got ", actions->scalar_type());
        a = solid(actions->to(at::kLong).reshape(-1));
    }
    if (valid) {
        type_check(valid->scalar_type() == at::kBool, "valid must be bool, got ", valid->scalar_type());
        v = rows_of(valid->sizes() == raw.sizes() ? *valid : valid->expand(raw.sizes()), A);
    }
    Tensor logp, entropy, top, top_logp;
    if (at::GradMode::is_enabled() && raw.requires_grad()) {
        const variable_list o = LogProbsNode::apply(flat, a, v, k);
        entropy = o[0];
        if (actions) logp = o[1];
        if (k) { top_logp = o[actions ? 2 : 1]; top = o[actions ? 3 : 2]; }
    } else {
        const LogProbs o = logprobs(flat, value(a), value(v), k, false);
        logp = o.logp; entropy = o.entropy; top = o.top; top_logp = o.top_logp;
    }
    const bool flatten = raw.dim() == 2;
    auto back = [&](const Tensor& t, bool wide) -> py::object {
        if (!t.defined()) return py::none();
        return py::cast(flatten ? t : wide ? t.view(with_last(lead, k)) : t.view(lead));
    };
    return py::make_tuple(back(logp, false), back(entropy, false), back(top, true), back(top_logp, true));
}

// ---- the residual stream between two blocks ----
enum Kind { NONE = BL_GATE_NONE, FULL = BL_GATE_FULL, CHANNEL = BL_GATE_CHANNEL, ROW = BL_GATE_ROW, PACKED };

struct GateArg { const void* p; int kind; long stride; };
GateArg gate_of(const Tensor& y, const Tensor& gate, int64_t kind, int64_t W) {
    if (kind == PACKED) return {ptr<char>(y) + W * y.element_size(), FULL, y.stride(0)};
    return {ptr(gate), (int)kind, kind == FULL || kind == ROW ? gate.stride(0) : 0};
}

struct Norm { Tensor out, h, stats; };
Norm norm_residual(const Tensor& x, const Tensor& y, const Tensor& alpha, const Tensor& post, const Tensor& gate, const Tensor& pre, int64_t kind, double eps,
                   at::ScalarType h_type, bool want_stats) {
    const int64_t R = x.size(0), W = x.size(1);
    const auto like = x.options().requires_grad(false);
    Norm o;
    if (y.defined()) o.out = at::empty({R, W}, like);
    if (pre.defined()) o.h = at::empty({R, W}, like.dtype(h_type));
    if (want_stats) o.stats = at::empty({R, 2}, like.dtype(at::kFloat));
    if (!R) return o;
    const GateArg g = gate_of(y, gate, kind, W);
    const c10::DeviceGuard guard(x.device());
    check(bl_norm_residual(ptr(x), code_of(x.scalar_type()), x.stride(0), ptr(y), code_of(h_type), row_stride(y), ptr<float>(alpha), ptr<float>(post), g.p, g.kind,
                           g.stride, ptr<float>(pre), (float)eps, R, (int)W, ptr(o.out), ptr(o.h), ptr<float>(o.stats), stream_of(x)));
    return o;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& y, const Maybe& alpha, const Maybe& post, const Maybe& gate, const Maybe& pre, int64_t kind,
                                 double eps, int64_t h_type) {
        const Norm o = norm_residual(x, value(y), value(alpha), value(post), value(gate), value(pre), kind, eps, (at::ScalarType)h_type, true);
        ctx->save_for_backward({x, value(y), value(alpha), value(post), value(gate), value(pre), o.stats});
        ctx->set_materialize_grads(false);
        ctx->saved_data["kind"] = kind; ctx->saved_data["eps"] = eps; ctx->saved_data["h_type"] = h_type;
        variable_list out;
        if (o.out.defined()) out.push_back(o.out);
        if (o.h.defined()) out.push_back(o.h);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once();
        const auto s = ctx->get_saved_variables();
        TORCH_CHECK(s[0].dim() == 2 && code_of(s[0].scalar_type()) >= 0, "a saved tensor came back from its hook with another shape or type");
        const int64_t kind = ctx->saved_data["kind"].toInt(), R = s[0].size(0), W = s[0].size(1);
        const at::ScalarType h_type = (at::ScalarType)ctx->saved_data["h_type"].toInt();
        kept(s[0], s[6], {R, W}, s[0].scalar_type());
        kept(s[1], s[0], {R, kind == PACKED ? 2 * W : W}, h_type); kept(s[2], s[0], {}, at::kFloat); kept(s[3], s[0], {W}, at::kFloat); kept(s[5], s[0], {W}, at::kFloat);
        if (kind == CHANNEL) kept(s[4], s[0], {W}, at::kFloat); else kept(s[4], s[0], {R, kind == ROW ? 1 : W}, h_type);
        kept(s[6], s[0], {R, 2}, at::kFloat);
        // (a saved-tensor hook may return them with other strides)
        auto rows = [](const Tensor& t) { return t.defined() && t.dim() == 2 ? rows_of(t, t.size(1)) : solid(t); };
        const Tensor x = rows(s[0]), y = rows(s[1]), alpha = plain(s[2]), post = solid(s[3]), gate = rows(s[4]), pre = solid(s[5]), stats = solid(s[6]);
        const Tensor g_out = y.defined() ? rows_of(g[0], W) : Tensor(), g_h = pre.defined() ? rows_of(g.back(), W) : Tensor();
        kept(g_out, x, {R, W}, x.scalar_type()); kept(g_h, x, {R, W}, h_type);
        auto like = [&](const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); };
        const Tensor dx = like(x), dy = like(y);
        Tensor dalpha = like(alpha), dpost = like(post), dgate = like(gate), dpre = g_h.defined() ? like(pre) : Tensor();
        if (!R) {
            for (Tensor* t : {&dalpha, &dpost, &dgate, &dpre}) if (t->defined()) t->zero_();
        } else {
            const GateArg ga = gate_of(y, gate, kind, W), gd = gate_of(dy, dgate, kind, W);
            const c10::DeviceGuard guard(x.device());
            const Tensor work = at::empty({bl_norm_residual_workspace(R, (int)W)}, x.options().dtype(at::kByte));
            check(bl_norm_residual_grad(ptr(x), code_of(x.scalar_type()), x.stride(0), ptr(y), code_of(h_type), row_stride(y), ptr<float>(alpha), ptr<float>(post), ga.p, ga.kind,
                                        ga.stride, ptr<float>(pre), (float)ctx->saved_data["eps"].toDouble(), R, (int)W, ptr<float>(stats), ptr(g_out), row_stride(g_out), ptr(g_h),
                                        row_stride(g_h), ptr(dx), ptr(dy), row_stride(dy), const_cast<void*>(gd.p), gd.stride, ptr<float>(dalpha), ptr<float>(dpost),
                                        ptr<float>(dpre), ptr(work), stream_of(x)));
        }
        return {dx, dy, dalpha, dpost, dgate, dpre, Tensor(), Tensor(), Tensor()};
    }
};

py::tuple py_norm_residual(const Tensor& x, const Maybe& y, const Maybe& alpha, const Maybe& post, const Maybe& gate, const Maybe& pre, double eps,
                           const std::optional<at::ScalarType>& dtype) {
    type_check(code_of(x.scalar_type()) >= 0, "x must be float32, float16 or bfloat16, got ", x.scalar_type());
    value_check(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= BL_NORM_MAX, "x must be (..., W) with W in 1 .. ", BL_NORM_MAX, ", got ", shape_of(x.sizes()));
    const Maybe x_ = x;
    transform_check("norm_residual", {&x_, &y, &alpha, &post, &gate, &pre});
    device_check(x, {&y, &alpha, &post, &gate, &pre});
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    const int64_t W = x.size(-1);
    if (!y) value_check(!alpha && !post && !gate && pre, "without y there is only h = pre * x / rms(x): alpha, post and gate must be None and pre given");
    else value_check(y->dim() == x.dim() && y->sizes().slice(0, y->dim() - 1) == lead && (y->size(-1) == W || y->size(-1) == 2 * W), "y must be ", shape_of(x.sizes()),
                     " or twice as wide, got ", shape_of(y->sizes()));
    const at::ScalarType h_type = y ? y->scalar_type() : dtype.value_or(x.scalar_type());
    type_check(h_type == x.scalar_type() || (x.scalar_type() == at::kFloat && code_of(h_type) >= 0),
               "y (or dtype) must be of x's type, or float16 / bfloat16 beside float32: got ", x.scalar_type(), " and ", h_type);
    type_check(!y || !dtype || *dtype == h_type, "h is of y's type");
    auto parameter = [&](const char* name, const Maybe& t, at::IntArrayRef shape) {
        if (t) value_check(t->sizes() == shape && t->scalar_type() == at::kFloat, name, " must be float32 of shape ", shape_of(shape), ", got ", t->scalar_type(), " ", shape_of(t->sizes()));
    };
    parameter("alpha", alpha, {}); parameter("post", post, {W}); parameter("pre", pre, {W});
    value_check(eps >= 0, "eps must not be negative, got ", eps);
    int64_t kind = NONE;
    if (y && y->size(-1) == 2 * W) {
        value_check(!gate, "y holds the gates already");
        kind = PACKED;
    } else if (gate) {
        kind = gate->dim() == 1 && gate->size(0) == W ? CHANNEL : gate->sizes() == x.sizes() ? FULL : gate->sizes() == at::IntArrayRef(with_last(lead, 1)) ? ROW : -1;
        value_check(kind >= 0, "gate must be ", shape_of({W}), ", ", shape_of(x.sizes()), " or ", shape_of(with_last(lead, 1)), ", got ", shape_of(gate->sizes()));
        type_check(gate->scalar_type() == (kind == CHANNEL ? at::kFloat : h_type), "a gate per channel is float32, any other of y's type: got ", gate->scalar_type());
    }
    const Tensor xs = rows_of(x, W), ys = y ? rows_of(*y, y->size(-1)) : Tensor(), al = plain(value(alpha)), po = solid(value(post)), pr = solid(value(pre));
    const Tensor gs = !gate ? Tensor() : kind == CHANNEL ? solid(*gate) : rows_of(*gate, gate->size(-1));
    Tensor out, h;
    if (at::GradMode::is_enabled() && (wants(x) || wants(ys) || wants(al) || wants(po) || wants(gs) || wants(pr))) {
        auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
        const variable_list o = NormNode::apply(xs, maybe(ys), maybe(al), maybe(po), maybe(gs), maybe(pr), kind, eps, (int64_t)h_type);
        if (y) out = o[0];
        if (pre) h = o.back();
    } else {
        const Norm o = norm_residual(xs, ys, al, po, gs, pr, kind, eps, h_type, false);
        out = o.out; h = o.h;
    }
    auto back = [&](const Tensor& t) -> py::object { return t.defined() ? py::cast(x.dim() == 2 ? t : t.view(x.sizes())) : py::object(py::none()); };
    return py::make_tuple(y ? back(out) : py::cast(x), back(h));
}

// ---- orthogonalisation ----
std::vector<Tensor> py_orthogonalize(const std::vector<Tensor>& mats, int64_t steps, double eps) {
    value_check(steps >= 1 && steps <= 1000, "steps must be in 1 .. 1000, got ", steps);
    value_check(eps >= 0, "eps must not be negative, got ", eps);
    const at::NoGradGuard no_grad;
    std::vector<Tensor> outs(mats.size()), solids(mats.size());
    for (size_t i = 0; i < mats.size(); i++) {
        const Tensor& m = mats[i];
        type_check(code_of(m.scalar_type()) >= 0, "matrices must be float32, float16 or bfloat16, got ", m.scalar_type());
        value_check(m.dim() == 2, "matrices must be two-dimensional, got ", shape_of(m.sizes()));
        value_check(m.size(0) <= BL_ORTHO_MAX && m.size(1) <= BL_ORTHO_MAX, "sides up to ", BL_ORTHO_MAX, " are supported, got ", shape_of(m.sizes()));
        const Maybe m_ = m;
        transform_check("orthogonalize", {&m_});
        device_check(m, {});
    }
    for (size_t i = 0; i < mats.size(); i++) {
        if (outs[i].defined()) continue;
        // this matrix and all behind it that go with it
        std::vector<const void*> in;
        std::vector<void*> out;
        const Tensor& m = mats[i];
        for (size_t j = i; j < mats.size(); j++) {
            const Tensor& o = mats[j];
            if (outs[j].defined() || o.sizes() != m.sizes() || o.scalar_type() != m.scalar_type() || o.device() != m.device()) continue;
            outs[j] = at::empty(o.sizes(), o.options().requires_grad(false));
            if (!o.numel()) continue;
            solids[j] = solid(o);
            in.push_back(solids[j].data_ptr()); out.push_back(outs[j].data_ptr());
        }
        if (in.empty()) continue;
        const c10::DeviceGuard guard(m.device());
        const int rows = (int)m.size(0), cols = (int)m.size(1), count = (int)in.size();
        const Tensor work = at::empty({bl_orthogonalize_workspace(count, rows, cols)}, m.options().dtype(at::kByte).requires_grad(false));
        check(bl_orthogonalize(in.data(), out.data(), count, code_of(m.scalar_type()), rows, cols, (int)steps, (float)eps, ptr(work), stream_of(m)));
    }
    return outs;
}

}  // namespace

PYBIND11_MODULE(_torchops, m) {
    m.def("logprobs", &py_logprobs);
    m.def("norm_residual", &py_norm_residual);
    m.def("orthogonalize", &py_orthogonalize);
}
