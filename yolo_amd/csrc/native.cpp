// Host side, in C++, of operators that are one or two short launches (Python module yolo_amd._native): allocation,
// launch and, where they are differentiable, the node of torch's autograd.  At small maps such a call is
// bound by the host.  A training step's node in Python costs it more than the kernels cost the GPU: its backward step runs on
// autograd's own thread, which has to take the interpreter's lock from the caller first.  Host time per call, in Python
// and here: group norm + Mish 13^2 x 1024 11.3 -> 6.0 us; with shortcut over 13^2 x 512, forward and backward, 116 -> 64-72; dropout
// with shortcut, forward and backward, 80 -> 50; 8-bit convolution 13^2 1024 -> 512 (one launch) 10.6 -> 8.1,
// 3x3 256 -> 512 (two) 17 -> 12.
//
// Arguments are checked by yolo_amd.training and yolo_amd.layers; the kernels are reached through the C entry points of
// the library that yolo_amd._lib has loaded, whose addresses it hands to init().
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/ymx.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

#define YMX_ENTRY_POINTS(X)                                                                                   \
    X(ymx_group_norm_workspace_bytes) X(ymx_group_norm_forward) X(ymx_group_norm_backward) X(ymx_dropout)        \
    X(ymx_conv2d_quantizes) X(ymx_quantized_bytes) X(ymx_quantize_blocks) X(ymx_conv2d_fused_ex) X(ymx_last_error)
struct {
#define X(name) decltype(&::name) name = nullptr;
    YMX_ENTRY_POINTS(X)
#undef X
} api;

// As yolo_amd._lib.check: what the entry points refuse is a ValueError.
void check(int rc) {
    if (rc == YMX_OK) return;
    const std::string text = api.ymx_last_error();
    if (rc == YMX_EARG || rc == YMX_EUNSUPPORTED) throw py::value_error("ymx: " + text);
    throw std::runtime_error("ymx (" + std::to_string(rc) + "): " + text);
}
void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
int dtype_of(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? YMX_BF16 : YMX_F32; }
Tensor dense(const Tensor &t, at::ScalarType type) { return (t.scalar_type() == type ? t : t.to(type)).contiguous(); }
Tensor cast(const Tensor &t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }
Tensor given(const optional<Tensor> &t) { return t ? *t : Tensor(); }
Tensor empty_as(const Tensor &t) { return at::empty(t.sizes(), t.options()); }
Tensor workspace(size_t bytes, const Tensor &like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }

// Whether a call over these tensors is recorded for back-propagation.  (Tangents are refused whether or not it is: a dual tensor
// need not require a gradient, and no_grad does not switch forward mode off.)
template <typename... Ts> bool records(const Ts &...t) {
    TORCH_CHECK(!(torch::autograd::isFwGradDefined(t) || ...), "yolo_amd.training: these operators have no forward-mode derivative");
    return at::GradMode::is_enabled() && (wants(t) || ...);
}
// A node whose gradients go to these tensors, in this order.
template <typename N, typename... Ts> std::shared_ptr<N> new_node(const Ts &...t) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(t...));
    return node;
}

// The gradients of a step that is itself being recorded (create_graph=True): an error for whoever differentiates them.
variable_list once(bool recorded, variable_list grads) {
    if (!recorded) return grads;
    variable_list in;
    for (const Tensor &g : grads)
        if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "yolo_amd.training: this operator is once_differentiable, its gradients cannot be differentiated again", (int64_t)in.size());
    variable_list out = (*error)(std::move(in));
    size_t n = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = out[n++];
    return grads;
}

// ---- group norm + activation + dropout + shortcut -----------------------------------------------------
struct GroupNormCall {
    long long B = 0, pix = 0;
    int C = 0, G = 0, act = 0, dtype = 0;
    double rate = 0.0;
    size_t ws = 0;
};
struct GroupNormOut {
    Tensor y, x, gamma, beta, stats;
    GroupNormCall call;
};
GroupNormOut gn_forward(const Tensor &x_in, const Tensor &gamma, const Tensor &beta, const optional<Tensor> &shortcut,
                        const optional<Tensor> &state, int64_t groups, int64_t act, double eps, double rate, bool keep) {
    GroupNormOut o;
    GroupNormCall &c = o.call;
    o.x = x_in.contiguous();
    o.gamma = dense(gamma, at::kFloat);
    o.beta = dense(beta, at::kFloat);
    o.y = empty_as(o.x);
    c.B = o.x.size(0);
    c.C = (int)o.x.size(-1);
    c.G = (int)groups;
    c.act = (int)act;
    c.dtype = dtype_of(o.x);
    c.rate = rate;
    if (keep) o.stats = at::empty({c.B, groups, 4}, o.gamma.options());
    if (o.x.numel() == 0) return o;                              // pix = 0: nothing is launched, here and backward
    c.pix = o.x.numel() / (c.B * c.C);
    c.ws = api.ymx_group_norm_workspace_bytes(c.B, c.pix, c.C, c.G);
    const c10::DeviceGuard guard(o.x.device());
    const Tensor sc = shortcut ? dense(*shortcut, o.x.scalar_type()) : Tensor(), ws = workspace(c.ws, o.x);
    check(api.ymx_group_norm_forward(o.x.data_ptr(), (const float *)o.gamma.data_ptr(), (const float *)o.beta.data_ptr(), address(sc), o.y.data_ptr(),
                         (float *)address(o.stats), c.B, c.pix, c.C, c.G, c.act, (float)eps, c.dtype, c.rate, state ? state->data_ptr() : nullptr,
                         ws.data_ptr(), c.ws, stream_of(o.x)));
    return o;
}

struct GroupNormBackward : Node {
    SavedVariable x_, gamma_, beta_, stats_, state_;
    GroupNormCall call;
    at::ScalarType gamma_type, beta_type, shortcut_type;

    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *v : {&x_, &gamma_, &beta_, &stats_, &state_}) v->reset_data();
    }
    // (The gradient of the shortcut is dy itself, not an alias of it: whoever accumulates it sees who else holds it.)
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        const bool recorded = at::GradMode::is_enabled();
        const at::AutoGradMode off(false);
        const Tensor x = x_.unpack(), gamma = gamma_.unpack(), beta = beta_.unpack(), stats = stats_.unpack(), state = state_.unpack();
        const bool need_x = task_should_compute_output(0), need_g = task_should_compute_output(1), need_b = task_should_compute_output(2);
        variable_list out(4);
        if (!grads[0].defined()) return out;
        if (need_x || need_g || need_b) {
            const Tensor dy = dense(grads[0], x.scalar_type());
            Tensor dx = empty_as(x), dgamma = empty_as(gamma), dbeta = empty_as(beta);
            if (call.pix > 0) {
                const c10::DeviceGuard guard(x.device());
                const Tensor ws = workspace(call.ws, x);
                check(api.ymx_group_norm_backward(x.data_ptr(), dy.data_ptr(), (const float *)gamma.data_ptr(), (const float *)beta.data_ptr(),
                                                  (const float *)stats.data_ptr(), dx.data_ptr(), (float *)dgamma.data_ptr(), (float *)dbeta.data_ptr(),
                                                  call.B, call.pix, call.C, call.G, call.act, call.dtype, call.rate, address(state), ws.data_ptr(),
                                                  call.ws, stream_of(x)));
            } else {
                dgamma.zero_();
                dbeta.zero_();
            }
            if (need_x) out[0] = dx;
            if (need_g) out[1] = cast(dgamma, gamma_type);
            if (need_b) out[2] = cast(dbeta, beta_type);
        }
        if (task_should_compute_output(3)) out[3] = cast(grads[0], shortcut_type);
        return once(recorded, std::move(out));
    }
};

Tensor group_norm_act(const Tensor &x, const Tensor &gamma, const Tensor &beta, const optional<Tensor> &shortcut, const optional<Tensor> &state,
                      int64_t groups, int64_t act, double eps, double rate) {
    const Tensor sc = given(shortcut);
    const bool recorded = records(x, gamma, beta, sc);
    GroupNormOut o;
    {
        const at::AutoGradMode off(false);
        o = gn_forward(x, gamma, beta, shortcut, state, groups, act, eps, rate, recorded);
    }
    if (recorded) {
        auto node = new_node<GroupNormBackward>(x, gamma, beta, sc);
        node->x_ = SavedVariable(o.x, false);
        node->gamma_ = SavedVariable(o.gamma, false);
        node->beta_ = SavedVariable(o.beta, false);
        node->stats_ = SavedVariable(o.stats, false);
        node->state_ = SavedVariable(given(state), false);
        node->call = o.call;
        node->gamma_type = gamma.scalar_type();
        node->beta_type = beta.scalar_type();
        node->shortcut_type = sc.defined() ? sc.scalar_type() : at::kFloat;
        torch::autograd::set_history(o.y, node);
    }
    return o.y;
}

// ---- dropout + shortcut ----------------------------------------------------------------------------------
Tensor dropout_run(const Tensor &x_in, const optional<Tensor> &shortcut, const Tensor &state, double rate) {
    const Tensor x = x_in.contiguous(), y = empty_as(x), sc = shortcut ? dense(*shortcut, x.scalar_type()) : Tensor();
    const c10::DeviceGuard guard(x.device());
    check(api.ymx_dropout(x.data_ptr(), address(sc), y.data_ptr(), x.numel(), dtype_of(x), rate, state.data_ptr(), stream_of(x)));
    return y;
}

struct DropoutBackward : Node {
    SavedVariable state_;
    at::ScalarType x_type, shortcut_type;
    double rate;

    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        state_.reset_data();
    }
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        const bool recorded = at::GradMode::is_enabled();
        const at::AutoGradMode off(false);
        const Tensor state = state_.unpack();
        variable_list out(2);
        if (!grads[0].defined()) return out;
        if (task_should_compute_output(0)) out[0] = dropout_run(cast(grads[0], x_type), std::nullopt, state, rate);
        if (task_should_compute_output(1)) out[1] = cast(grads[0], shortcut_type);
        return once(recorded, std::move(out));
    }
};

Tensor dropout(const Tensor &x, const optional<Tensor> &shortcut, const Tensor &state, double rate) {
    const Tensor sc = given(shortcut);
    const bool recorded = records(x, sc);
    Tensor y;
    {
        const at::AutoGradMode off(false);
        y = dropout_run(x, shortcut, state, rate);
    }
    if (recorded) {
        auto node = new_node<DropoutBackward>(x, sc);
        node->state_ = SavedVariable(state, false);
        node->x_type = x.scalar_type();
        node->shortcut_type = sc.defined() ? sc.scalar_type() : at::kFloat;
        node->rate = rate;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---- convolution block in 8 bits ----------------------------------------------------------------------------
// t: the map, or (quantised) the buffer of a quantised one; out: the result's place, pixel stride out_ld, or nothing.
Tensor conv8(const Tensor &t, bool quantised, int64_t B, int64_t H, int64_t W, int64_t cin, const Tensor &packed, const optional<Tensor> &scale,
             const optional<Tensor> &shift, const optional<Tensor> &residual, const optional<Tensor> &out, int64_t out_ld, int64_t k,
             int64_t stride, int64_t oh, int64_t ow, int64_t cout, int64_t act, bool fp32) {
    const at::AutoGradMode off(false);
    const c10::DeviceGuard guard(t.device());
    void *stream = stream_of(t);
    const auto aligned = [](const Tensor &v) { return ((uintptr_t)v.data_ptr() & 15) == 0 ? v : v.clone(); };
    const at::ScalarType type = fp32 ? at::kFloat : at::kBFloat16;
    const Tensor y = out ? *out : at::empty({B, oh, ow, cout}, t.options().dtype(type));
    const Tensor res = residual ? aligned(dense(*residual, type)) : Tensor();
    Tensor x = t;
    int x_type = YMX_F8E4M3;
    if (!quantised) {
        x = aligned(t.contiguous());
        if (x.scalar_type() == at::kBFloat16 && api.ymx_conv2d_quantizes(B * oh * ow, (int)cout, (int)k, fp32 ? YMX_F32 : YMX_BF16)) {
            x_type = YMX_BF16;                                   // few pixels: by the layer's own kernel
        } else {
            const Tensor q = workspace(api.ymx_quantized_bytes(B * H * W, (int)cin), x);
            check(api.ymx_quantize_blocks(x.data_ptr(), q.data_ptr(), B * H * W, (int)cin, dtype_of(x), 0, stream));
            x = q;
        }
    }
    check(api.ymx_conv2d_fused_ex(x.data_ptr(), packed.data_ptr(), scale ? scale->data_ptr() : nullptr, shift ? shift->data_ptr() : nullptr,
                                  address(res), y.data_ptr(), (int)B, (int)H, (int)W, (int)cin, (int)cout, (int)k, (int)stride, (int)act,
                                  YMX_F8E4M3, x_type, fp32 ? YMX_F32 : YMX_BF16, 0, 0, (int)out_ld, stream));
    return y;
}

std::vector<std::string> entry_points() {
    return {
#define X(name) #name,
        YMX_ENTRY_POINTS(X)
#undef X
    };
}
void init(const std::unordered_map<std::string, uintptr_t> &addresses) {
#define X(name) api.name = (decltype(api.name))addresses.at(#name);
    YMX_ENTRY_POINTS(X)
#undef X
}

}  // namespace

PYBIND11_MODULE(_native, m) {
    m.attr("ENTRY_POINTS") = entry_points();
    m.def("init", &init);
    m.def("group_norm_act", &group_norm_act);
    m.def("dropout", &dropout);
    m.def("conv8", &conv8);
}
