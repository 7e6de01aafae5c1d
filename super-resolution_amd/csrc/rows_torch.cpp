// PyTorch side of the row operators (srmi/rows.py): argument checks, output and workspace tensors, and the autograd nodes, over the
// C ABI of include/srmi.h.  C++ because a row operator can be a 3 us kernel: the same nodes written in Python cost 18 us more in the
// forward call and as much again in the backward one.
//
// Workspaces are tensors of the call: nothing is shared between streams, graphs or threads.
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <mutex>
#include <tuple>
#include <unordered_set>

#include "../../include/srmi.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct SrmiFailure : std::runtime_error {
    int code;
    SrmiFailure(int c, const char* msg) : std::runtime_error(msg), code(c) {}
};
void check(int rc) {
    if (rc) throw SrmiFailure(rc, srmi_last_error());
}

int dtype_code(const Tensor& t) {
    if (t.scalar_type() == at::kFloat) return SRMI_F32;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "srmi supports float32 and bfloat16 storage, got ", t.scalar_type());
    return SRMI_BF16;
}
void require_cuda(const Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), "srmi: ", what, " is on ", t.device(),
                "; the HIP kernels need a ROCm device tensor (there is deliberately no CPU fallback)");
}
void check_like(const Tensor& t, const char* what, at::ScalarType dtype, const Tensor& x, at::IntArrayRef shape) {
    require_cuda(t, what);
    TORCH_CHECK_TYPE(t.scalar_type() == dtype, "srmi.rows: ", what, " is ", t.scalar_type(), ", expected ", dtype);
    TORCH_CHECK_VALUE(t.device() == x.device(), "srmi.rows: ", what, " is on ", t.device(), ", x on ", x.device());
    TORCH_CHECK_VALUE(t.sizes() == shape, "srmi.rows: ", what, " has shape ", t.sizes(), ", expected ", shape);
}
int check_x(const Tensor& x) {
    require_cuda(x, "input");
    TORCH_CHECK_VALUE(x.dim() >= 1, "srmi.rows: x needs at least one axis");
    return dtype_code(x);
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
// A tangent of forward-mode AD would be lost: the operators have no such formula, and a result without a tangent passes for a constant.
void check_tangents(std::initializer_list<const Tensor*> operands) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "srmi.rows: forward-mode automatic differentiation is not supported");
}
// The dispatcher sees the allocations of a call and no operator, and the kernels read the operands' own storage.  What records calls to run
// them again (torch.jit.trace, make_fx, torch.export) would replay an output nobody writes, and a wrapper tensor (FakeTensor,
// DTensor) has no storage of its own: both are refused.  Modes that only watch (FlopCounterMode) or keep and recompute
// (selective checkpointing) get correct results and are let through.
void check_recorders(std::initializer_list<const Tensor*> operands) {
    typedef c10::impl::TorchDispatchModeKey Mode;
    bool recording = torch::jit::tracer::isTracing();
    for (Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL}) recording |= c10::impl::TorchDispatchModeTLS::get_mode(m).has_value();
    TORCH_CHECK_NOT_IMPLEMENTED(!recording, "srmi.rows: the operators cannot be traced or exported, a replay would return memory that nobody wrote");
    for (const Tensor* t : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize})),
                                    "srmi.rows: a tensor subclass with its own dispatch has no storage that a kernel can read");
}
// autograd counts the tensors a node was given, not its optional arguments
typedef std::optional<Tensor> Opt;
Opt opt(const Tensor& t) { return t.defined() ? Opt(t) : std::nullopt; }
constexpr char ONCE[] = "srmi.rows: the backward passes are not differentiable themselves";
void once(const Tensor& dy) {
    check_recorders({&dy});
    check_tangents({&dy});
    TORCH_CHECK(!(at::GradMode::is_enabled() && dy.requires_grad()), ONCE);
}
// A gradient that depends on tensors that require one themselves: under create_graph=True differentiating it raises, instead of
// passing for a constant.
void once_more(Tensor& g, bool depends) {
    if (!g.defined() || !depends || !at::GradMode::is_enabled()) return;
    torch::autograd::DelayedError node(ONCE, 1);
    g = node.apply({g.detach().requires_grad_()})[0];
}

// Saved-tensor hooks decide what a backward pass gets back: another layout is as good (torch.autograd.graph.save_on_cpu hands back dense rows
// for strided ones), so strides come from the restored tensor, never from the forward pass; another type, place or shape
// is refused, since the kernels would read past it.
void check_restored(const Tensor& t, const char* what, at::ScalarType dtype, at::Device device, at::IntArrayRef shape) {
    TORCH_CHECK(t.device() == device && t.scalar_type() == dtype && t.sizes() == shape, "srmi.rows: a saved-tensor hook handed back ", what,
                " as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", saved was ", dtype, " ", shape, " on ", device);
}

// A backward pass that is captured must not meet a node that was made on the default stream: an operation before the capture, or a leaf's
// accumulation node that an eager graph, still alive, refers to.  Autograd would make that stream wait for the capturing one, which
// the default stream cannot, and the process ends.  (Another stream, such as the one of warm-up runs whose last graph is still
// referred to, joins the capture and is fine.)  Looked for in the operands and in everything they were computed from.
void check_capture(std::initializer_list<const Tensor*> operands) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    auto push = [&](std::shared_ptr<torch::autograd::Node> node) {
        if (node && seen.insert(node.get()).second) todo.push_back(std::move(node));
    };
    for (const Tensor* t : operands)
        if (wants_grad(*t)) push(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        const auto node = todo.back();
        todo.pop_back();
        const auto stream = node->stream();
        TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(stream->device_index()).id(),
                    "srmi.rows: graph capture over a leaf that an eager autograd graph of the default stream still refers to; delete that graph first");
        for (const auto& edge : node->next_edges()) push(edge.function);
    }
}

// Kernels read what lies in memory: a view that negates it (the imaginary part of a conjugate) is written out first.
Tensor as_stored(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return t.defined() ? as_stored(t).contiguous() : t; }

// `t` as [rows, last axis]: in place if the last axis is dense and the leading ones walk with one stride, else a copy
std::tuple<Tensor, int64_t> strided_rows(const Tensor& view) {
    const Tensor t = as_stored(view);
    const int64_t c = t.size(-1);
    if (t.is_contiguous()) return {t, c};
    if (t.stride(-1) == 1 || c <= 1) {
        int64_t ld = -1, n = 1;
        bool uniform = true;
        for (int64_t i = t.dim() - 2; i >= 0 && uniform; --i) {
            if (t.size(i) == 1) continue;
            if (ld < 0) ld = t.stride(i);
            else uniform = t.stride(i) == ld * n;
            n *= t.size(i);
        }
        if (ld < 0) ld = c;
        if (uniform && ld >= std::max<int64_t>(c, 1)) return {t, ld};
    }
    return {t.contiguous(), c};
}
int align_of(std::initializer_list<const Tensor*> ts) {
    uintptr_t bits = 0;
    for (const Tensor* t : ts) bits |= (uintptr_t)ptr(*t);
    return bits & 15 ? 0 : 16;
}

// ---- linear --------------------------------------------------------------------------------------------------------------
size_t linear_ws(const srmi_linear_desc& d, int pass) {
    size_t n = 0;
    check(srmi_linear_workspace_bytes(&d, pass, &n));
    return n;
}

struct LinearOut { Tensor y, z, x, w; };

LinearOut linear_run(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int act, float param, bool want_z) {
    const int64_t N = w.size(0), K = w.size(1);
    LinearOut o;
    int64_t ldx, ldw, ldr = 0;
    std::tie(o.x, ldx) = strided_rows(x);
    std::tie(o.w, ldw) = strided_rows(w);
    Tensor rr;
    if (r.defined()) std::tie(rr, ldr) = strided_rows(r);
    const Tensor bb = dense(b);
    auto shape = x.sizes().vec();
    int64_t M = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) M *= shape[i];
    shape.back() = N;
    o.y = at::empty(shape, x.options());
    if (want_z) o.z = at::empty({M, N}, x.options().dtype(x.scalar_type() == at::kBFloat16 ? at::kHalf : at::kFloat));
    if (M == 0 || N == 0) return o;
    TORCH_CHECK_VALUE(N <= INT32_MAX && K <= INT32_MAX, "srmi.rows.linear: more than 2^31 features");
    const srmi_linear_desc d = {M, (int32_t)N, (int32_t)K, dtype_code(x), act, param, align_of({&o.x, &o.w}), ldx, ldw, ldr, 0};
    const size_t bytes = linear_ws(d, SRMI_PASS_FWD);
    const Tensor ws = workspace(bytes, x);
    check(srmi_linear_fwd(&d, ptr(o.x), ptr(o.w), ptr(bb), ptr(rr), ptr(o.y), ptr(o.z), ptr(ws), bytes, stream_of(x)));
    return o;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& ob, const Opt& orr, int64_t act, double param) {
        const Tensor b = ob.value_or(Tensor()), r = orr.value_or(Tensor());
        const bool need = wants_grad(x) || wants_grad(w) || wants_grad(b);
        // ReLU and LeakyReLU keep the sign of z: without a residual on top y itself is enough for the backward pass
        const bool by_sign = !r.defined() && (act == SRMI_ACT_RELU || (act == SRMI_ACT_LRELU && param > 0.0));
        const bool slope = act != SRMI_ACT_NONE && need;
        LinearOut o = linear_run(x, w, b, r, (int)act, (float)param, slope && !by_sign);
        ctx->save_for_backward({wants_grad(w) ? o.x : Tensor(), wants_grad(x) ? o.w : Tensor(), slope ? (by_sign ? o.y : o.z) : Tensor()});
        ctx->saved_data["act"] = act;
        ctx->saved_data["param"] = param;
        ctx->saved_data["xshape"] = x.sizes().vec();
        ctx->saved_data["N"] = w.size(0);
        ctx->saved_data["K"] = w.size(1);
        ctx->saved_data["need"] = (int64_t)(wants_grad(x) | wants_grad(w) << 1 | wants_grad(b) << 2 | wants_grad(r) << 3);
        ctx->saved_data["by_sign"] = by_sign;
        ctx->saved_data["res"] = (int64_t)(2 + b.defined());                    // the residual's place among the tensors
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& dy = grads[0];
        once(dy);
        const auto saved = ctx->get_saved_variables();
        const int64_t N = ctx->saved_data["N"].toInt(), K = ctx->saved_data["K"].toInt(), need = ctx->saved_data["need"].toInt();
        const auto xshape = ctx->saved_data["xshape"].toIntVector();
        int64_t M = 1;
        for (size_t i = 0; i + 1 < xshape.size(); ++i) M *= xshape[i];
        if (saved[0].defined()) check_restored(saved[0], "linear's x", dy.scalar_type(), dy.device(), xshape);
        if (saved[1].defined()) check_restored(saved[1], "linear's weight", dy.scalar_type(), dy.device(), {N, K});
        if (saved[2].defined()) {
            if (ctx->saved_data["by_sign"].toBool()) check_restored(saved[2], "linear's output", dy.scalar_type(), dy.device(), dy.sizes());
            else check_restored(saved[2], "linear's pre-activation", dy.scalar_type() == at::kBFloat16 ? at::kHalf : at::kFloat, dy.device(), {M, N});
        }
        // of the inputs that require a gradient, those that this backward pass was asked for
        auto asked = [&](int i) { return (need >> i & 1) && ctx->needs_input_grad(i < 3 ? i : ctx->saved_data["res"].toInt()); };
        Tensor dx, dw, db;
        if (asked(0) || asked(1) || asked(2)) {
            const c10::OptionalDeviceGuard guard(dy.device());
            Tensor dyr, x, w;
            int64_t lddy, ldx = K, ldw = K;
            std::tie(dyr, lddy) = strided_rows(dy);
            if (saved[0].defined()) std::tie(x, ldx) = strided_rows(saved[0]);
            if (saved[1].defined()) std::tie(w, ldw) = strided_rows(saved[1]);
            const Tensor s = dense(saved[2]);
            if (asked(0)) dx = at::empty(xshape, dy.options());
            if (asked(1)) dw = at::empty({N, K}, dy.options());
            if (asked(2)) db = at::empty({N}, dy.options());
            const srmi_linear_desc d = {M, (int32_t)N, (int32_t)K, dtype_code(dy), (int32_t)ctx->saved_data["act"].toInt(),
                                        (float)ctx->saved_data["param"].toDouble(), align_of({&x, &w, &dyr}), ldx, ldw, 0, lddy};
            const size_t bytes = linear_ws(d, SRMI_PASS_BWD);
            const Tensor ws = workspace(bytes, dy);
            check(srmi_linear_bwd(&d, ptr(x), ptr(w), ptr(s), ptr(dyr), ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream_of(dy)));
            const bool slope = d.act != SRMI_ACT_NONE;
            once_more(dx, slope || (need & 2));
            once_more(dw, slope || (need & 1));
            once_more(db, slope);
        }
        return {dx, dw, db, asked(3) ? dy : Tensor(), Tensor(), Tensor()};
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const Opt& bias, const Opt& residual, int64_t act, double param) {
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    check_recorders({&x, &w, &b, &r});
    check_tangents({&x, &w, &b, &r});
    check_x(x);
    TORCH_CHECK_VALUE(w.dim() == 2, "srmi.rows.linear: weight must be [out_features, in_features]");
    check_like(w, "weight", x.scalar_type(), x, w.sizes());
    TORCH_CHECK_VALUE(x.size(-1) == w.size(1), "srmi.rows.linear: x has ", x.size(-1), " features, weight ", w.sizes());
    if (b.defined()) check_like(b, "bias", x.scalar_type(), x, {w.size(0)});
    if (r.defined()) {
        auto shape = x.sizes().vec();
        shape.back() = w.size(0);
        check_like(r, "residual", x.scalar_type(), x, shape);
    }
    const c10::OptionalDeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b) || wants_grad(r))) {
        check_capture({&x, &w, &b, &r});
        return LinearFn::apply(x, w, opt(b), opt(r), act, param);
    }
    return linear_run(x, w, b, r, (int)act, (float)param, false).y;
}

// ---- layer norm ------------------------------------------------------------------------------------------------------------
int param_code(const Tensor& w, const Tensor& b) { return w.defined() ? dtype_code(w) : b.defined() ? dtype_code(b) : SRMI_F32; }

struct NormOut { Tensor y, stats, x; };

NormOut norm_run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool keep) {
    const int64_t C = x.size(-1), rows = x.numel() / C;
    auto [xr, ldx] = strided_rows(x);
    Tensor y = at::empty(x.sizes(), x.options()), stats;
    if (keep) stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    if (rows) {
        TORCH_CHECK_VALUE(C <= INT32_MAX, "srmi.rows.layer_norm: more than 2^31 features");
        const Tensor wc = dense(w), bc = dense(b);
        const srmi_norm_desc d = {rows, (int32_t)C, dtype_code(x), param_code(w, b), (float)eps, ldx, 0};
        float* st = (float*)ptr(stats);
        check(srmi_layer_norm_fwd(&d, ptr(xr), ptr(wc), ptr(bc), ptr(y), st, keep ? st + rows : nullptr, stream_of(x)));
    }
    return {y, stats, xr};
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& ow, const Opt& ob, double eps) {
        const Tensor w = ow.value_or(Tensor()), b = ob.value_or(Tensor());
        NormOut o = norm_run(x, w, b, eps, true);
        ctx->save_for_backward({o.x, w, o.stats});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["xshape"] = x.sizes().vec();
        ctx->saved_data["param"] = (int64_t)param_code(w, b);
        ctx->saved_data["need"] = (int64_t)(wants_grad(x) | wants_grad(w) << 1 | wants_grad(b) << 2);
        ctx->saved_data["bias"] = (int64_t)(1 + w.defined());                   // the bias's place among the tensors
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& dy = grads[0];
        once(dy);
        const auto saved = ctx->get_saved_variables();
        const auto xshape = ctx->saved_data["xshape"].toIntVector();
        const int64_t C = xshape.back(), rows = dy.numel() / C, need = ctx->saved_data["need"].toInt();
        const int pcode = (int)ctx->saved_data["param"].toInt();
        check_restored(saved[0], "layer_norm's x", dy.scalar_type(), dy.device(), xshape);
        check_restored(saved[2], "layer_norm's statistics", at::kFloat, dy.device(), {2, rows});
        if (saved[1].defined()) check_restored(saved[1], "layer_norm's weight", pcode == SRMI_F32 ? at::kFloat : at::kBFloat16, dy.device(), {C});
        auto asked = [&](int i) { return (need >> i & 1) && ctx->needs_input_grad(i < 2 ? i : ctx->saved_data["bias"].toInt()); };
        const c10::OptionalDeviceGuard guard(dy.device());
        const auto [xr, ldx] = strided_rows(saved[0]);
        const auto [dyr, lddy] = strided_rows(dy);
        const Tensor stats = dense(saved[2]), w = dense(saved[1]);
        const auto popt = dy.options().dtype(pcode == SRMI_F32 ? at::kFloat : at::kBFloat16);
        Tensor dx = asked(0) ? at::empty(xshape, dy.options()) : Tensor(), dw = asked(1) ? at::empty({C}, popt) : Tensor();
        const Tensor db = asked(2) ? at::empty({C}, popt) : Tensor();
        const srmi_norm_desc d = {rows, (int32_t)C, dtype_code(dy), pcode, (float)ctx->saved_data["eps"].toDouble(), ldx, lddy};
        size_t bytes = 0;
        if (dw.defined() || db.defined()) check(srmi_layer_norm_workspace_bytes(&d, &bytes));
        const Tensor ws = workspace(bytes, dy);
        const float* st = (const float*)ptr(stats);
        check(srmi_layer_norm_bwd(&d, ptr(xr), ptr(w), st, st + rows, ptr(dyr), ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream_of(dy)));
        once_more(dx, true);
        once_more(dw, need & 1);
        return {dx, dw, db, Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, const Opt& weight, const Opt& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    check_recorders({&x, &w, &b});
    check_tangents({&x, &w, &b});
    check_x(x);
    const int64_t C = x.size(-1);
    TORCH_CHECK_VALUE(C > 0, "srmi.rows.layer_norm: the last axis is empty");
    TORCH_CHECK_VALUE(eps >= 0.0, "srmi.rows.layer_norm: eps must be >= 0");
    const Tensor& p = w.defined() ? w : b;
    const at::ScalarType pt = p.defined() && p.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type();
    if (w.defined()) check_like(w, "weight", pt, x, {C});
    if (b.defined()) check_like(b, "bias", pt, x, {C});
    const c10::OptionalDeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) {
        check_capture({&x, &w, &b});
        return LayerNormFn::apply(x, opt(w), opt(b), eps);
    }
    return norm_run(x, w, b, eps, false).y;
}

// ---- dropout ---------------------------------------------------------------------------------------------------------------
Tensor dropout_run(const Tensor& x_, const Tensor& residual, double p, uint64_t seed, uint64_t offset, const Tensor& rng) {
    const Tensor x = dense(x_), r = dense(residual);
    Tensor y = at::empty(x.sizes(), x.options());
    if (x.numel())
        check(srmi_dropout(ptr(x), ptr(r), ptr(y), (size_t)x.numel(), dtype_code(x), p, seed, offset, (const uint64_t*)ptr(rng), stream_of(x)));
    return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& orr, double p, int64_t seed, int64_t offset, const Opt& orng) {
        const Tensor r = orr.value_or(Tensor()), rng = orng.value_or(Tensor());
        ctx->save_for_backward({rng});              // an in-place write between the passes would change the mask: torch reports it
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["need"] = (int64_t)(wants_grad(x) | wants_grad(r) << 1);
        return dropout_run(x, r, p, (uint64_t)seed, (uint64_t)offset, rng);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& dy = grads[0];
        once(dy);
        Tensor rng = ctx->get_saved_variables()[0];
        if (rng.defined()) {
            check_restored(rng, "dropout's [seed, offset]", at::kLong, dy.device(), {2});
            rng = dense(rng);
        }
        const int64_t need = ctx->saved_data["need"].toInt();
        auto asked = [&](int i) { return (need >> i & 1) && ctx->needs_input_grad(i); };
        const c10::OptionalDeviceGuard guard(dy.device());
        Tensor dx;
        if (asked(0))
            dx = dropout_run(dy, Tensor(), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                             (uint64_t)ctx->saved_data["offset"].toInt(), rng);
        return {dx, asked(1) ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x, const Opt& residual, double p, uint64_t seed, uint64_t offset, const Opt& device_rng) {
    const Tensor r = residual.value_or(Tensor()), rng = device_rng.value_or(Tensor());
    check_recorders({&x, &r, &rng});
    check_tangents({&x, &r});
    check_x(x);
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "srmi.rows.dropout: p must be in [0, 1], got ", p);
    if (rng.defined()) {
        check_like(rng, "seed", at::kLong, x, {2});
        TORCH_CHECK_VALUE(rng.is_contiguous(), "srmi.rows.dropout: the [seed, offset] tensor must be contiguous");
    }
    if (r.defined()) check_like(r, "residual", x.scalar_type(), x, x.sizes());
    const c10::OptionalDeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(r))) {
        check_capture({&x, &r});
        return DropoutFn::apply(x, opt(r), p, (int64_t)seed, (int64_t)offset, opt(rng));
    }
    return dropout_run(x, r, p, seed, offset, rng);
}

}  // namespace

PYBIND11_MODULE(_rows, m) {
    py::register_exception_translator([](std::exception_ptr e) {
        try {
            if (e) std::rethrow_exception(e);
        } catch (const SrmiFailure& f) {
            const py::object type = py::module_::import("srmi._lib").attr("SrmiError");
            PyErr_SetObject(type.ptr(), type(f.code, f.what()).ptr());
        }
    });
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("linear", &linear, nogil);
    m.def("layer_norm", &layer_norm, nogil);
    m.def("dropout", &dropout, nogil);
    m.def("strided_rows", &strided_rows, nogil);
}
