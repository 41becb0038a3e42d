// The dense linear layer and layer norm as differentiable PyTorch operations over the C ABI: argument checks, allocation
// and the two autograd nodes. They are C++ because of what a call costs besides its kernels: a small training step of a
// layer took 114 to 123 us with the nodes in Python (89 us of that for any Python node, forward and backward), a small
// call without gradients 10 us.
//
// Every call runs on x's device and PyTorch's current stream there (the backward pass on the forward pass's, as PyTorch's
// engine sets it) and allocates with PyTorch's allocator, workspaces too, so calls may overlap on several streams and be
// captured into CUDA graphs. Refused arguments raise ValueError or TypeError, forward-mode tangents and traces
// NotImplementedError, a refused launch RuntimeError.

#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "weightferry_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

template <typename... Args>
[[noreturn]] void refuse_value(const Args &...args) {
    throw py::value_error(c10::str(args...));
}
template <typename... Args>
[[noreturn]] void refuse_type(const Args &...args) {
    throw py::type_error(c10::str(args...));
}

void check(int rc, const char *what) {
    TORCH_CHECK(rc == WF_OK, what, ": weightferry_b200 status ", rc, " (", wf_status_string(rc), ")");
}

wf_stream_t stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

int code_of(at::ScalarType t) { return t == at::kHalf ? WF_F16 : t == at::kBFloat16 ? WF_BF16 : WF_F32; }

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *mut(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

bool wants_grad(const MaybeTensor &t) { return t.has_value() && t->requires_grad(); }

// t [rows, cols] with a row's values side by side, and its row pitch
std::pair<Tensor, int64_t> as_rows(const Tensor &t) {
    const int64_t rows = t.size(0), cols = t.size(1), s0 = rows == 1 ? cols : t.stride(0);
    if ((t.stride(1) != 1 && cols > 1) || s0 < cols) return {t.contiguous(), cols};
    return {t, s0};
}

// An operand of a product as TMA reads it: 16-byte aligned, a pitch of a multiple of 8 values. Other layouts (odd widths,
// slices) are to be copied.
struct Operand {
    Tensor t;
    int64_t ld = 0;
    wf_copy_rows copy = {};
};

Operand as_operand(const Tensor &t) {
    const int64_t rows = t.size(0), cols = t.size(1), s0 = rows == 1 ? up8(cols) : t.stride(0);
    if ((t.stride(1) == 1 || cols == 1) && s0 % 8 == 0 && s0 >= cols && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0)
        return {t, s0};
    Operand o{at::empty({rows, up8(cols)}, t.options()), up8(cols)};
    o.copy = {t.const_data_ptr(), o.t.mutable_data_ptr(), t.stride(0), o.ld, rows, cols};
    return o;
}

// x's and w's operands (either may be undefined), their copies in one launch
std::pair<Operand, Operand> as_operands(const Tensor &x, const Tensor &w) {
    const Tensor *given[2] = {&x, &w};
    Operand out[2];
    Tensor rows[2];  // live until the copies are launched
    wf_copy_rows copies[2];
    int n = 0;
    for (int i = 0; i < 2; ++i) {
        if (!given[i]->defined()) continue;
        int64_t ld;
        std::tie(rows[i], ld) = as_rows(*given[i]);
        out[i] = as_operand(rows[i]);
        if (out[i].copy.dst != nullptr) copies[n] = out[i].copy, copies[n++].ld_src = ld;
    }
    if (n > 0) check(wf_copy_rows16(copies, n, stream_of(x.defined() ? x : w)), "wf_copy_rows16");
    return {out[0], out[1]};
}

// A saved tensor as the graph gives it back. Hooks (save_on_cpu, checkpoints, a user's own) return a tensor of their own:
// its strides and address are its own too, so a pitch is taken from it and never kept beside it. Its shape, type and device
// must be what was saved.
void check_saved(const char *what, const Tensor &t, at::IntArrayRef shape, at::ScalarType type, const at::Device &device) {
    TORCH_CHECK(t.sizes() == shape && t.scalar_type() == type && t.device() == device, what, ": a saved tensor of shape ", shape,
                ", ", type, " on ", device, " came back as ", t.sizes(), ", ", t.scalar_type(), " on ", t.device());
}

// rows of x for each row of p ([n] or [groups, n]): as given, or all m rows divided evenly
int64_t group_rows(const char *what, const Tensor &p, int64_t m, const std::optional<int64_t> &given) {
    const int64_t groups = p.dim() == 1 ? 1 : p.size(0);
    if (!given.has_value()) {
        if (m % groups) refuse_value(what, ": ", groups, " rows do not divide ", m, " rows; give rows_per_group");
        return std::max<int64_t>(1, m / groups);
    }
    if (*given < 1 || (m && groups != (m - 1) / *given + 1))
        refuse_value(what, ": ", groups, " rows for ", m, " rows in groups of ", *given);
    return *given;
}

// What a gradient depends on, when it is itself recorded (create_graph): raises for whoever asks how.
struct Refusal : public torch::autograd::Node {
    explicit Refusal(torch::autograd::edge_list &&next) : Node(std::move(next)) {}
    variable_list apply(variable_list &&) override { TORCH_CHECK(false, "this gradient cannot be differentiated again"); }
};

// Ties the fresh gradients of a recorded backward pass to dy and to everything that the forward pass was given, so that no way
// of differentiating them finds them constant.
void only_once(variable_list &grads, const Tensor &dy) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list next{torch::autograd::impl::gradient_edge(dy)};
    if (const auto node = torch::autograd::get_current_node())
        next.insert(next.end(), node->next_edges().begin(), node->next_edges().end());
    std::shared_ptr<Refusal> refusal;
    for (const Tensor &g : grads) {
        if (!g.defined() || g.is_same(dy)) continue;  // the residual's gradient is dy
        if (refusal == nullptr) refusal = std::shared_ptr<Refusal>(new Refusal(std::move(next)), torch::autograd::deleteNode);
        torch::autograd::set_history(g, refusal);
    }
}

// Tangents and traces, which the operations would drop without a word: their outputs come out of kernels that neither sees.
void refuse_unseen(const char *what, std::initializer_list<const Tensor *> tensors) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !Modes::get_mode(Key::PROXY) && !Modes::get_mode(Key::FAKE), what,
                                ": a call cannot be traced");
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(t == nullptr || !t->_fw_grad(0).defined(), what, ": no forward-mode derivatives");
}

// ------------------------------------------------------------------------------------------------ dense linear layer
struct LinearCall {
    int64_t act, rpg, m, n, k;
};

struct Kept {  // what the backward pass may need: x and w as the products read them, z [m, up8(n)]
    Tensor x, w, z;
};

Tensor linear_forward(const Tensor &x, const Tensor &w, const MaybeTensor &bias, const MaybeTensor &resid,
                      const MaybeTensor &gate, const LinearCall &c, std::optional<at::ScalarType> z_type, Kept *kept) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = c.n;
    Tensor y = at::empty(shape, x.options());
    if (c.m == 0 || c.n == 0) return y;
    const auto [xo, wo] = as_operands(x.dim() == 2 ? x : x.reshape({c.m, c.k}), w);
    wf_linear_args a = {};
    Tensor b, g, r, z;
    if (bias) b = bias->contiguous();
    if (gate) g = gate->contiguous();
    if (resid) std::tie(r, a.ld_resid) = as_rows(resid->dim() == 2 ? *resid : resid->reshape({c.m, c.n}));
    if (z_type) {
        z = at::empty({c.m, up8(c.n)}, x.options().dtype(*z_type));
        a.z = z.mutable_data_ptr();
        a.ldz = up8(c.n);
        a.z_type = code_of(*z_type);
    }
    a.x = xo.t.const_data_ptr(), a.w = wo.t.const_data_ptr(), a.bias = ptr(b), a.gate = ptr(g), a.resid = ptr(r);
    a.y = y.mutable_data_ptr();
    a.ldx = xo.ld, a.ldw = wo.ld, a.ldy = c.n, a.rows_per_group = c.rpg, a.m = c.m, a.n = c.n, a.k = c.k;
    a.act = static_cast<int32_t>(c.act), a.type = code_of(x.scalar_type());
    check(wf_linear(&a, stream_of(x)), "wf_linear");
    if (kept != nullptr) *kept = Kept{xo.t, wo.t, z};
    return y;
}

struct LinearNode : public torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const MaybeTensor &bias,
                          const MaybeTensor &resid, const MaybeTensor &gate, const LinearCall &c) {
        const bool need_x = x.requires_grad(), need_w = w.requires_grad(), need_b = wants_grad(bias), need_g = wants_grad(gate);
        // How z is kept. The activation's slope is constant where f16 ends, so f16 (clamped, 11 bits) keeps it more exactly
        // than bf16 would. The gate's gradient reads activation(z) itself: exactly (f32), or in a bf16 layer without an
        // activation as that layer rounds it (two bytes a value less to write and read). f16 does not hold every z of a finite
        // gate * z.
        std::optional<at::ScalarType> z_type;
        if (need_g) z_type = c.act || x.scalar_type() == at::kHalf ? at::kFloat : x.scalar_type();
        else if (c.act && (need_x || need_w || need_b)) z_type = at::kHalf;
        Kept kept;
        Tensor y = linear_forward(x, w, bias, resid, gate, c, z_type, &kept);
        ctx->save_for_backward({need_w ? kept.x : Tensor(), need_x ? kept.w : Tensor(),
                                gate && (need_x || need_w || need_b) ? *gate : Tensor(), kept.z});
        std::vector<int64_t> d{c.act, c.rpg, c.m, c.n, c.k, c.m && c.n ? kept.x.size(1) : 0, c.m && c.n ? kept.w.size(1) : 0, need_x, need_w, need_b, wants_grad(resid), need_g,
                               gate ? gate->dim() : 0, gate ? gate->size(0) : 0,
                               z_type ? static_cast<int64_t>(*z_type) : 0};
        d.insert(d.end(), x.sizes().begin(), x.sizes().end());
        ctx->saved_data["call"] = std::move(d);
        return y;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const std::vector<int64_t> d = ctx->saved_data["call"].toIntVector();
        const int64_t act = d[0], rpg = d[1], m = d[2], n = d[3], k = d[4];
        const bool need_x = d[7], need_w = d[8], need_b = d[9], need_r = d[10], need_g = d[11];
        const Tensor &dy = grads[0];
        const variable_list saved = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(dy.device());
        const auto opt = dy.options();
        auto fresh = [&](bool need, at::IntArrayRef shape) {
            return !need ? Tensor() : m && n ? at::empty(shape, opt) : at::zeros(shape, opt);
        };
        const std::vector<int64_t> gate_shape = d[12] == 2 ? std::vector<int64_t>{d[13], n} : std::vector<int64_t>{n};
        variable_list out{fresh(need_x, at::IntArrayRef(d).slice(15)), fresh(need_w, {n, k}), fresh(need_b, {n}),
                          need_r ? dy : Tensor(), fresh(need_g, gate_shape), Tensor()};
        if (m && n && (need_x || need_w || need_b || need_g)) {
            const at::AutoGradMode off(false);
            const auto [dy2, lddy] = as_rows(dy.dim() == 2 ? dy : dy.reshape({m, n}));
            wf_linear_grad_args a = {};
            const at::ScalarType type = dy.scalar_type();
            Tensor gate, z;
            if (saved[0].defined()) check_saved("linear: x", saved[0], {m, d[5]}, type, dy.device());
            if (saved[1].defined()) check_saved("linear: weight", saved[1], {n, d[6]}, type, dy.device());
            if (saved[2].defined()) {
                check_saved("linear: gate", saved[2], gate_shape, type, dy.device());
                gate = saved[2].contiguous();
            }
            if (saved[3].defined()) {
                check_saved("linear: the pre-activation", saved[3], {m, up8(n)}, static_cast<at::ScalarType>(d[14]), dy.device());
                std::tie(z, a.ldz) = as_rows(saved[3]);
            }
            const auto [xo, wo] = as_operands(saved[0], saved[1]);
            a.dy = dy2.const_data_ptr(), a.x = ptr(xo.t), a.w = ptr(wo.t), a.z = ptr(z), a.gate = ptr(gate);
            a.dx = mut(out[0]), a.dw = mut(out[1]), a.db = mut(out[2]), a.dg = mut(out[4]);
            a.lddy = lddy, a.ldx = xo.ld, a.ldw = wo.ld, a.lddx = k, a.lddw = k, a.rows_per_group = rpg;
            a.m = m, a.n = n, a.k = k, a.act = static_cast<int32_t>(act), a.type = code_of(type);
            a.z_type = z.defined() ? code_of(z.scalar_type()) : 0;
            a.workspace_bytes = wf_linear_backward_needs(&a);
            const Tensor work = a.workspace_bytes ? at::empty({a.workspace_bytes}, opt.dtype(at::kByte)) : Tensor();
            a.workspace = mut(work);
            check(wf_linear_backward(&a, stream_of(dy)), "wf_linear_backward");
        }
        only_once(out, dy);
        return out;
    }
};

constexpr const char *kActivations[] = {"none", "relu", "silu", "gelu", "gelu_tanh"};  // the codes WF_ACT_*

Tensor linear(const Tensor &x, const Tensor &weight, const MaybeTensor &bias, const std::string &activation,
              const MaybeTensor &residual, const MaybeTensor &gate, const std::optional<int64_t> &rows_per_group) {
    refuse_unseen("linear", {&x, &weight, bias ? &*bias : nullptr, residual ? &*residual : nullptr, gate ? &*gate : nullptr});
    const at::ScalarType t = x.scalar_type();
    if (t != at::kBFloat16 && t != at::kHalf) refuse_type("linear: x is ", t, "; bfloat16 or float16 is needed");
    int64_t act = 0;
    while (act < 5 && activation != kActivations[act]) ++act;
    if (act == 5) refuse_value("linear: activation '", activation, "' is not one of none, relu, silu, gelu, gelu_tanh");
    const std::pair<const char *, const Tensor *> rest[] = {{"weight", &weight}, {"bias", bias ? &*bias : nullptr},
                                                            {"residual", residual ? &*residual : nullptr},
                                                            {"gate", gate ? &*gate : nullptr}};
    for (const auto &[name, p] : rest)
        if (p != nullptr && p->scalar_type() != t) refuse_type("linear: ", name, " is ", p->scalar_type(), ", x is ", t);
    if (x.dim() < 1 || weight.dim() != 2 || x.size(-1) != weight.size(1))
        refuse_value("linear: x ", x.sizes(), " and weight ", weight.sizes(), " do not match");
    LinearCall c{act, 1, 0, weight.size(0), weight.size(1)};
    if (c.k < 1) refuse_value("linear: a layer without inputs");
    c.m = x.numel() / c.k;
    if (bias && (bias->dim() != 1 || bias->size(0) != c.n)) refuse_value("linear: bias ", bias->sizes(), " for ", c.n, " outputs");
    if (residual && (residual->dim() != x.dim() || residual->size(-1) != c.n ||
                     residual->sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1)))
        refuse_value("linear: residual ", residual->sizes(), " for x ", x.sizes(), " and ", c.n, " outputs");
    c.rpg = std::max<int64_t>(1, c.m);
    if (gate) {
        if ((gate->dim() != 1 && gate->dim() != 2) || gate->size(-1) != c.n || (gate->dim() == 2 && gate->size(0) == 0))
            refuse_value("linear: gate ", gate->sizes(), " for ", c.n, " outputs");
        c.rpg = group_rows("linear: gate", *gate, c.m, rows_per_group);
    } else if (rows_per_group) {
        refuse_value("linear: rows_per_group without a gate");
    }
    for (const auto &[name, p] : rest)
        if (p != nullptr && p->device() != x.device()) refuse_value("linear: ", name, " is on ", p->device(), ", x on ", x.device());
    if (!x.is_cuda()) refuse_value("linear: x is on ", x.device(), "; a CUDA device is needed");
    const c10::cuda::CUDAGuard guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants_grad(bias) || wants_grad(residual) ||
                                       wants_grad(gate)))
        return LinearNode::apply(x, weight, bias, residual, gate, c);
    return linear_forward(x, weight, bias, residual, gate, c, std::nullopt, nullptr);
}

// -------------------------------------------------------------------------------------------------------- layer norm
struct NormCall {
    int64_t rpg, m, d;
    double eps;
};

struct Stats {
    Tensor x, stats;  // x's rows [m, d]; mean and rstd [2, m]
};

Tensor norm_forward(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, const NormCall &c, Stats *kept) {
    Tensor y = at::empty(x.sizes(), x.options());
    if (c.m == 0) return y;
    const auto [x2, ldx] = as_rows(x.dim() == 2 ? x : x.reshape({c.m, c.d}));
    wf_layer_norm_args a = {};
    Tensor w, b, stats;
    a.type = a.w_type = code_of(x.scalar_type());
    if (bias) b = bias->contiguous(), a.w_type = code_of(b.scalar_type());
    if (weight) w = weight->contiguous(), a.w_type = code_of(w.scalar_type());
    if (kept != nullptr) {
        stats = at::empty({2, c.m}, x.options().dtype(at::kFloat));
        a.mean = stats.mutable_data_ptr<float>();
        a.rstd = a.mean + c.m;
        *kept = Stats{x2, stats};
    }
    a.x = x2.const_data_ptr(), a.w = ptr(w), a.b = ptr(b), a.y = y.mutable_data_ptr();
    a.ldx = ldx, a.ldy = c.d, a.rows = c.m, a.d = c.d, a.rows_per_group = c.rpg, a.eps = static_cast<float>(c.eps);
    check(wf_layer_norm(&a, stream_of(x)), "wf_layer_norm");
    return y;
}

struct NormNode : public torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias,
                          const NormCall &c) {
        Stats kept;
        Tensor y = norm_forward(x, weight, bias, c, &kept);
        ctx->save_for_backward({kept.x, weight ? *weight : Tensor(), kept.stats});
        const Tensor p = weight ? *weight : bias ? *bias : Tensor();
        std::vector<int64_t> d{c.rpg, c.m, c.d, x.requires_grad(), wants_grad(weight), wants_grad(bias),
                               p.defined() ? static_cast<int64_t>(p.scalar_type()) : 0, p.defined() ? p.dim() : 0};
        if (p.defined()) d.insert(d.end(), p.sizes().begin(), p.sizes().end());
        d.insert(d.end(), x.sizes().begin(), x.sizes().end());
        ctx->saved_data["call"] = std::move(d);
        return y;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const std::vector<int64_t> v = ctx->saved_data["call"].toIntVector();
        const int64_t rpg = v[0], m = v[1], d = v[2];
        const Tensor &dy = grads[0];
        const variable_list saved = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(dy.device());
        const auto opt = dy.options();
        const auto p_opt = opt.dtype(static_cast<at::ScalarType>(v[6]));
        const at::IntArrayRef p_shape = at::IntArrayRef(v).slice(8, v[7]), x_shape = at::IntArrayRef(v).slice(8 + v[7]);
        auto fresh = [&](bool need, at::IntArrayRef shape, const at::TensorOptions &o) {
            return !need ? Tensor() : m ? at::empty(shape, o) : at::zeros(shape, o);
        };
        variable_list out{fresh(v[3], x_shape, opt), fresh(v[4], p_shape, p_opt), fresh(v[5], p_shape, p_opt), Tensor()};
        if (m && (v[3] || v[4] || v[5])) {
            const at::AutoGradMode off(false);
            const auto [dy2, lddy] = as_rows(dy.dim() == 2 ? dy : dy.reshape({m, d}));
            wf_layer_norm_grad_args a = {};
            a.type = code_of(dy.scalar_type());
            a.w_type = v[7] ? code_of(static_cast<at::ScalarType>(v[6])) : a.type;
            Tensor work;
            if (v[4] || v[5]) {
                a.workspace_bytes = wf_layer_norm_backward_workspace(m, d, rpg, a.type);
                work = at::empty({a.workspace_bytes}, opt.dtype(at::kByte));
            }
            check_saved("layer_norm: x", saved[0], {m, d}, dy.scalar_type(), dy.device());
            check_saved("layer_norm: the statistics", saved[2], {2, m}, at::kFloat, dy.device());
            if (saved[1].defined())
                check_saved("layer_norm: weight", saved[1], p_shape, static_cast<at::ScalarType>(v[6]), dy.device());
            const Tensor w = saved[1].defined() ? saved[1].contiguous() : Tensor(), stats = saved[2].contiguous();
            const auto [x2, ldx] = as_rows(saved[0]);
            a.dy = dy2.const_data_ptr(), a.x = x2.const_data_ptr(), a.w = ptr(w);
            a.mean = stats.const_data_ptr<float>(), a.rstd = a.mean + m;
            a.dx = mut(out[0]), a.dw = mut(out[1]), a.db = mut(out[2]), a.workspace = mut(work);
            a.lddy = lddy, a.ldx = ldx, a.lddx = d, a.rows = m, a.d = d, a.rows_per_group = rpg;
            check(wf_layer_norm_backward(&a, stream_of(dy)), "wf_layer_norm_backward");
        }
        only_once(out, dy);
        return out;
    }
};

Tensor layer_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps,
                  const std::optional<int64_t> &rows_per_group) {
    refuse_unseen("layer_norm", {&x, weight ? &*weight : nullptr, bias ? &*bias : nullptr});
    const at::ScalarType t = x.scalar_type();
    if (t != at::kBFloat16 && t != at::kHalf && t != at::kFloat)
        refuse_type("layer_norm: x is ", t, "; bfloat16, float16 or float32 is needed");
    if (x.dim() < 1 || x.size(-1) < 1) refuse_value("layer_norm: x ", x.sizes(), " has no values to normalise");
    if (!(eps >= 0)) refuse_value("layer_norm: eps ", eps);
    NormCall c{1, 0, x.size(-1), eps};
    c.m = x.numel() / c.d;
    c.rpg = std::max<int64_t>(1, c.m);
    const Tensor *p = weight ? &*weight : bias ? &*bias : nullptr;
    if (p != nullptr) {
        for (const auto &[name, q] : {std::pair<const char *, const MaybeTensor *>{"weight", &weight}, {"bias", &bias}}) {
            if (!q->has_value()) continue;
            const Tensor &u = **q;
            if ((u.scalar_type() != t && u.scalar_type() != at::kFloat) || u.scalar_type() != p->scalar_type())
                refuse_type("layer_norm: ", name, " is ", u.scalar_type(), "; ", t, " or float32 is needed, weight and bias alike");
            if ((u.dim() != 1 && u.dim() != 2) || u.size(-1) != c.d || u.sizes() != p->sizes() || u.size(0) == 0)
                refuse_value("layer_norm: ", name, " ", u.sizes(), " for rows of ", c.d);
            if (u.device() != x.device()) refuse_value("layer_norm: ", name, " is on ", u.device(), ", x on ", x.device());
        }
        c.rpg = group_rows("layer_norm: weight", *p, c.m, rows_per_group);
    } else if (rows_per_group) {
        refuse_value("layer_norm: rows_per_group without weight or bias");
    }
    if (!x.is_cuda()) refuse_value("layer_norm: x is on ", x.device(), "; a CUDA device is needed");
    const c10::cuda::CUDAGuard guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias)))
        return NormNode::apply(x, weight, bias, c);
    return norm_forward(x, weight, bias, c, nullptr);
}

}  // namespace

PYBIND11_MODULE(wf_torch, m) {
    // wrapped: PyTorch's own errors keep their types, an allocation that fails is a torch.OutOfMemoryError
    m.def("linear", torch::wrap_pybind_function(&linear));
    m.def("layer_norm", torch::wrap_pybind_function(&layer_norm));
}
