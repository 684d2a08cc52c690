// torch's side of the operators over fp32, bf16 and fp16 tensors (mpgnn_layer_norm_*,
// mpgnn_grouped_linear_*, mpgnn_clip_*): argument checks, outputs and workspaces from torch's allocator,
// autograd nodes, and the calls of the C ABI on torch's current stream. Nothing is computed here.
//
// This is C++ because a step's small calls are bound by the host: autograd runs the backward of GPU tensors
// on a thread of its own, where Python costs three times what it costs in the caller's. operators.py loads
// the module at its first call; it links libmpgnn_rgcn.so, the library that _lib.py has checked and loaded.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

#include "mpgnn_rgcn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int32_t dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MPGNN_F32;
        case at::kBFloat16: return MPGNN_BF16;
        case at::kHalf: return MPGNN_F16;
        default: return -1;
    }
}

int32_t require(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "mpgnn_amd: `", name, "` is on ", t.device(),
                "; the operators run only as HIP kernels on a ROCm GPU (there is no CPU fallback). Move the model and "
                "data to 'cuda'.");
    const int32_t code = dtype_code(t);
    TORCH_CHECK_TYPE(code >= 0, "mpgnn_amd: `", name, "` must be float32, bfloat16 or float16, got ", t.scalar_type());
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, "mpgnn_amd: `", name, "` must be dense, got ", t.layout());
    return code;
}

// A tangent of forward-mode differentiation would be dropped, and a trace would record the outputs' allocation
// without the kernel that fills them: both are refused. (Not where forward mode is off, as it is inside the forward
// of a torch.autograd.Function, which answers for the derivative itself.)
void refuse_tangent(const Tensor& t, const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode() ||
                                    !t._fw_grad(/*level=*/0).defined(),
                                "mpgnn_amd: ", what, " has no forward-mode derivative: an argument carries a tangent");
}

void refuse_tracing(const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                                "mpgnn_amd: ", what, " cannot be recorded by torch.jit.trace or make_fx");
}

void refuse_transforms(const char* what, const Tensor& a, const Tensor& b = {}, const Tensor& c = {}) {
    refuse_tracing(what);
    refuse_tangent(a, what);
    refuse_tangent(b, what);
    refuse_tangent(c, what);
}

// The C entry points' statuses as the exceptions that _lib.check raises for them.
void check(int32_t status, const char* what) {
    if (status == MPGNN_OK) return;
    const std::string text = std::string(what) + ": " + mpgnn_last_error();
    TORCH_CHECK_VALUE(status != MPGNN_ERR_ARG, text);
    TORCH_CHECK_NOT_IMPLEMENTED(status != MPGNN_ERR_UNSUPPORTED, text);
    TORCH_CHECK(false, text);
}

// The device of the call made current (a launch goes to the current device) and torch's stream on it.
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream()) {}
};

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// A view that negates its memory (the imaginary part of a conjugate) is written out: kernels read memory.
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

Tensor dense(const Tensor& t) { return as_stored(t).contiguous(); }

// A tensor as rows of its last dimension: itself where its rows lie a constant pitch apart (contiguous,
// or a column slice of a matrix), else a contiguous copy.
struct Rows {
    Tensor t;
    int64_t rows, pitch;
    explicit Rows(const Tensor& given) : t(as_stored(given)) {
        const Tensor& x = t;
        const int64_t width = x.size(-1);
        rows = x.dim() == 2 ? x.size(0) : x.numel() / width;
        pitch = width;
        if (x.is_contiguous()) return;
        if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= width) pitch = x.stride(0);
        else t = t.contiguous();
    }
};

// An argument that may be left out, as an autograd node takes it.
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// The operators are differentiable once: where a graph of the backward is asked for, the gradients raise
// when that graph is run backward, whatever it would have been differentiated by.
variable_list once(variable_list out, const char* what) {
    if (!at::GradMode::is_enabled()) return out;
    for (Tensor& t : out)
        if (t.defined()) t = t.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("mpgnn_amd: ") + what + " has no second derivative", static_cast<int64_t>(out.size()));
    return (*error)(std::move(out));
}

// Which of an operator's tensor arguments want a gradient, as bits.
int64_t wanted(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    return wants_grad(x) | wants_grad(weight) << 1 | wants_grad(bias) << 2;
}

// ---------------------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------------------
struct NormTypes {
    int32_t x, w;
};

Tensor norm_forward(const Rows& x, const Tensor& weight, const Tensor& bias, double eps, NormTypes ty, const Tensor& like,
                    Tensor* stats) {
    Tensor y = at::empty_like(like, at::MemoryFormat::Contiguous);
    float* mean = nullptr;
    if (stats) {
        *stats = at::empty({2, x.rows}, like.options().dtype(at::kFloat));
        mean = stats->data_ptr<float>();
    }
    On on(like);
    check(mpgnn_layer_norm_fwd(x.t.data_ptr(), x.rows, like.size(-1), x.pitch, ty.x, data(weight), data(bias), ty.w, eps,
                               y.data_ptr(), mean, mean ? mean + x.rows : nullptr, on.stream),
          "mpgnn_layer_norm_fwd");
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w,
                          const std::optional<Tensor>& b, double eps, int64_t xcode, int64_t wcode) {
        const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
        const Rows r(x);
        Tensor stats;
        Tensor y = norm_forward(r, weight, bias, eps, {(int32_t)xcode, (int32_t)wcode}, x, &stats);
        ctx->save_for_backward({r.t, weight, stats});
        ctx->saved_data["types"] = xcode * 16 + wcode;
        ctx->saved_data["want"] = wanted(x, weight, bias);
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_tangent(grads[0], "layer_norm");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        const int64_t types = ctx->saved_data["types"].toInt(), want = ctx->saved_data["want"].toInt();
        const NormTypes ty{(int32_t)(types / 16), (int32_t)(types % 16)};
        const Rows r(x), d(grads[0]);
        const int64_t width = x.size(-1);
        const auto params = x.options().dtype(ty.w == ty.x ? x.scalar_type() : at::kFloat);
        Tensor dx, dw, db, ws;
        if (want & 1) dx = at::empty_like(x, at::MemoryFormat::Contiguous);
        if (want & 2) dw = at::empty({width}, params);
        if (want & 4) db = at::empty({width}, params);
        if (dw.defined() || db.defined()) {
            int64_t n = 0;
            check(mpgnn_layer_norm_bwd_workspace_bytes(r.rows, width, &n), "mpgnn_layer_norm_bwd_workspace_bytes");
            ws = bytes(std::max<int64_t>(n, 16), x);  // of its own per call: a captured one stays in its graph's pool
        }
        const float* mean = stats.data_ptr<float>();
        On on(x);
        check(mpgnn_layer_norm_bwd(d.t.data_ptr(), d.pitch, r.t.data_ptr(), r.pitch, r.rows, width, ty.x, data(weight),
                                   ty.w, mean, mean + r.rows, data(dx), data(dw), data(db), data(ws), on.stream),
              "mpgnn_layer_norm_bwd");
        variable_list out = once({dx, dw, db}, "layer_norm");
        out.resize(6);  // eps and the types have no gradient
        return out;
    }
};

int32_t norm_param(const Tensor& p, const char* name, const Tensor& x, int32_t code) {
    const int32_t c = require(p, name);
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == x.size(-1), "`", name, "` has shape ", p.sizes(), ", expected [",
                      x.size(-1), "]");
    TORCH_CHECK(p.device() == x.device(), "`", name, "` is on ", p.device(), ", x on ", x.device());
    TORCH_CHECK_TYPE(c == code || c == MPGNN_F32, "`", name, "` must be ", x.scalar_type(), " or Float, got ",
                     p.scalar_type());
    return c;
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
    refuse_transforms("layer_norm", x, weight.value_or(Tensor()), bias.value_or(Tensor()));
    const int32_t code = require(x, "x");
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0,
                      "layer_norm normalises a last dimension of at least one element, got shape ", x.sizes());
    int32_t wcode = code;
    Tensor w, b;
    if (weight) {
        wcode = norm_param(*weight, "weight", x, code);
        w = dense(*weight);
    }
    if (bias) {
        const int32_t c = norm_param(*bias, "bias", x, code);
        TORCH_CHECK_TYPE(!weight || c == wcode, "weight and bias must have one type, got ", weight->scalar_type(), " and ",
                         bias->scalar_type());
        wcode = c;
        b = dense(*bias);
    }
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(b)))
        return LayerNorm::apply(x, given(w), given(b), eps, (int64_t)code, (int64_t)wcode);
    return norm_forward(Rows(x), w, b, eps, {code, wcode}, x, nullptr);
}

// ---------------------------------------------------------------------------------------
// grouped linear
// ---------------------------------------------------------------------------------------
Tensor grouped_forward(const Rows& x, const Tensor& weight, const Tensor& bias, const Tensor& ptr) {
    Tensor y = at::empty({x.rows, weight.size(2)}, x.t.options());
    On on(x.t);
    check(mpgnn_grouped_linear_fwd(x.t.data_ptr(), x.rows, x.pitch, dtype_code(x.t), weight.data_ptr(), weight.size(0),
                                   weight.size(1), weight.size(2), data(bias), ptr.data_ptr(),
                                   ptr.scalar_type() == at::kLong ? 64 : 32, y.data_ptr(), on.stream),
          "mpgnn_grouped_linear_fwd");
    return y;
}

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& b,
                          const Tensor& ptr) {
        const Tensor bias = b.value_or(Tensor());
        const Rows r(x);
        const Tensor w = dense(weight);
        ctx->save_for_backward({r.t, w, ptr});
        ctx->saved_data["want"] = wanted(x, weight, bias);
        return grouped_forward(r, w, bias.defined() ? dense(bias) : bias, ptr);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_tangent(grads[0], "grouped_linear");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &ptr = saved[2];
        const Rows r(x), d(grads[0]);
        const int64_t groups = w.size(0), k = w.size(1), n = w.size(2), want = ctx->saved_data["want"].toInt();
        const int32_t code = dtype_code(x), bits = ptr.scalar_type() == at::kLong ? 64 : 32;
        Tensor dx, dw, db, ws;
        On on(x);
        if (want & 1) {
            dx = at::empty({r.rows, k}, x.options());
            check(mpgnn_grouped_linear_dgrad(d.t.data_ptr(), r.rows, d.pitch, code, w.data_ptr(), groups, k, n,
                                             ptr.data_ptr(), bits, dx.data_ptr(), on.stream),
                  "mpgnn_grouped_linear_dgrad");
        }
        if (want & 6) {
            dw = at::empty({groups, k, n}, x.options());
            if (want & 4) db = at::empty({groups, n}, x.options());
            int64_t size = 0;
            check(mpgnn_grouped_linear_wgrad_workspace_bytes(r.rows, groups, k, n, &size),
                  "mpgnn_grouped_linear_wgrad_workspace_bytes");
            if (size) ws = bytes(size, x);
            check(mpgnn_grouped_linear_wgrad(r.t.data_ptr(), r.pitch, d.t.data_ptr(), d.pitch, r.rows, code, groups, k, n,
                                             ptr.data_ptr(), bits, dw.data_ptr(), data(db), data(ws), on.stream),
                  "mpgnn_grouped_linear_wgrad");
        }
        variable_list out = once({dx, want & 2 ? dw : Tensor(), db}, "grouped_linear");
        out.resize(4);  // group_ptr has no gradient
        return out;
    }
};

Tensor grouped_linear(const Tensor& x, const Tensor& weight, const Tensor& ptr, const std::optional<Tensor>& bias) {
    refuse_transforms("grouped_linear", x, weight, bias.value_or(Tensor()));
    const int32_t code = require(x, "x");
    TORCH_CHECK_VALUE(x.dim() == 2 && weight.dim() == 3 && ptr.dim() == 1,
                      "grouped_linear takes x [rows, K], weight [groups, K, N] and group_ptr [groups + 1], got ",
                      x.sizes(), ", ", weight.sizes(), " and ", ptr.sizes());
    const int64_t groups = weight.size(0), k = weight.size(1), n = weight.size(2);
    TORCH_CHECK_VALUE(groups > 0 && k > 0 && n > 0,
                      "grouped_linear needs at least one group, input and output column, got weight ", weight.sizes());
    TORCH_CHECK(x.size(1) == k, "mat1 and mat2 shapes cannot be multiplied (", x.size(0), "x", x.size(1), " and ", k, "x",
                n, ")");
    TORCH_CHECK_VALUE(ptr.size(0) == groups + 1, "group_ptr has ", ptr.size(0), " entries, expected groups + 1 = ",
                      groups + 1);
    TORCH_CHECK_TYPE(ptr.scalar_type() == at::kLong || ptr.scalar_type() == at::kInt,
                     "group_ptr must be int32 or int64, got ", ptr.scalar_type());
    TORCH_CHECK_TYPE(require(weight, "weight") == code, "`weight` must be ", x.scalar_type(), " as x is, got ", weight.scalar_type());
    TORCH_CHECK(weight.device() == x.device(), "`weight` is on ", weight.device(), ", x on ", x.device());
    TORCH_CHECK(ptr.device() == x.device(), "`group_ptr` is on ", ptr.device(), ", x on ", x.device());
    Tensor b;
    if (bias) {
        TORCH_CHECK_TYPE(require(*bias, "bias") == code, "`bias` must be ", x.scalar_type(), " as x is, got ", bias->scalar_type());
        TORCH_CHECK(bias->device() == x.device(), "`bias` is on ", bias->device(), ", x on ", x.device());
        TORCH_CHECK_VALUE(bias->dim() == 2 && bias->size(0) == groups && bias->size(1) == n, "bias has shape ",
                          bias->sizes(), ", expected [", groups, ", ", n, "]");
        b = *bias;
    }
    const Tensor p = ptr.contiguous();
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants_grad(b)))
        return GroupedLinear::apply(x, weight, given(b), p);
    return grouped_forward(Rows(x), dense(weight), b.defined() ? dense(b) : b, p);
}

// ---------------------------------------------------------------------------------------
// global norm and clipping
// ---------------------------------------------------------------------------------------
enum Scaled { NONE = 0, OUT = 1, IN_PLACE = 2 };

// The norm of `grads`, and the scaled tensors: none, in `outs` (new ones if there is no list), or in the
// gradients themselves (strided ones and views that negate are copied, and copied back).
std::pair<Tensor, std::vector<Tensor>> clip(const std::vector<Tensor>& grads, std::optional<std::vector<Tensor>> outs,
                                            int64_t scaled, double max_norm, bool largest) {
    const bool in_place = scaled == IN_PLACE, fresh = scaled == OUT && !outs;
    const char* what = in_place ? "gradients" : "tensors";
    refuse_tracing("clipping");
    const size_t n = grads.size();
    const Tensor& first = grads[0];
    std::vector<mpgnn_clip_tensor> records(n);
    std::vector<Tensor> to;                           // given or made: where the scaled tensors go
    if (outs) to = std::move(*outs);
    std::vector<Tensor> copies;                       // of gradients that are not dense
    std::vector<std::pair<size_t, size_t>> back;      // (gradient, its copy) to be written back
    for (size_t i = 0; i < n; ++i) {
        const Tensor& g = grads[i];
        refuse_tangent(g, "clipping");
        mpgnn_clip_tensor& r = records[i];
        r.dtype = require(g, what);
        TORCH_CHECK(g.device() == first.device(), what, " are on several devices: ", first.device(), " and ", g.device());
        r.numel = g.numel();
        if (g.is_contiguous() && !g.is_neg()) {
            r.grad = g.data_ptr();
        } else {
            if (in_place)
                for (int64_t d = 0; d < g.dim(); ++d)
                    TORCH_CHECK_VALUE(g.stride(d) != 0 || g.size(d) < 2,
                                      "a gradient is an expanded tensor, whose elements share memory: it cannot be scaled "
                                      "in place");
            copies.push_back(dense(g.detach()));
            if (in_place) back.emplace_back(i, copies.size() - 1);
            r.grad = copies.back().data_ptr();
        }
        if (in_place) {
            r.out = const_cast<void*>(r.grad);
        } else if (fresh) {
            to.push_back(at::empty(g.sizes(), g.options()));
            r.out = to.back().data_ptr();
        } else if (scaled) {
            const Tensor& o = to[i];
            refuse_tangent(o, "clipping");
            TORCH_CHECK_VALUE(o.is_cuda() && o.scalar_type() == g.scalar_type() && o.sizes() == g.sizes() &&
                                  o.device() == g.device() && o.layout() == at::kStrided && o.is_contiguous() && !o.is_neg(),
                              "out must hold contiguous tensors of the inputs' sizes, types and device");
            r.out = o.data_ptr();
        }
    }
    // the C entry point refuses tensors that overlap, but of a strided gradient it sees the copy
    if (!back.empty()) {
        std::vector<const void*> written;
        for (const Tensor& g : grads)
            if (g.numel()) written.push_back(g.data_ptr());
        std::sort(written.begin(), written.end());
        TORCH_CHECK_VALUE(std::adjacent_find(written.begin(), written.end()) == written.end(),
                          "one tensor is to be scaled twice");
    }
    int64_t size = 0;
    check(mpgnn_clip_workspace_bytes((int32_t)n, &size), "mpgnn_clip_workspace_bytes");
    const Tensor ws = bytes(size, first);
    Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
    On on(first);
    check(mpgnn_clip_by_global_norm(records.data(), (int32_t)n, largest ? MPGNN_NORM_INF : MPGNN_NORM_2, max_norm,
                                    norm.data_ptr<float>(), ws.data_ptr(), on.stream),
          "mpgnn_clip_by_global_norm");
    if (scaled && !fresh) {
        at::NoGradGuard no_grad;
        for (const auto& [i, c] : back) grads[i].copy_(copies[c]);
        // written behind autograd's back, as any in-place operator counts
        for (const Tensor& t : in_place ? grads : to)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    return {norm, std::move(to)};
}

}  // namespace

PYBIND11_MODULE(_operators, m) {
    // without the GIL, and torch's errors as the Python exceptions they stand for
    m.def("layer_norm", torch::wrap_pybind_function_no_gil(layer_norm));
    m.def("grouped_linear", torch::wrap_pybind_function_no_gil(grouped_linear));
    m.def("clip", torch::wrap_pybind_function_no_gil(clip));
}
