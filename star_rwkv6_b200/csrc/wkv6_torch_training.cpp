// Native call path of the losses on given tokens (loss.py) and of the AdamW step (optim.py): one C++ function per call.
//
// The small calls are bound by the host: a policy update of 66 tokens is 10 us of kernels and took 180 us through Python (argument
// checks, ctypes structs, a Python autograd node), a step over 52 small tensors 260 us for 8 us of kernel.  Every function here
// returns None when the call is not the plain one it handles; the Python path then runs, and raises the error where there is one.
#include "wkv6_torch.h"

#include <c10/cuda/CUDAGraphsC10Utils.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <vector>

namespace wkv6_native {

namespace {

struct Api {
    decltype(&::wkv6_token_log_probs) token_log_probs = nullptr;
    decltype(&::wkv6_token_log_probs_backward) token_log_probs_backward = nullptr;
    decltype(&::wkv6_capture_id) capture_id = nullptr;
    decltype(&::wkv6_policy_loss) policy_loss = nullptr;
    decltype(&::wkv6_policy_loss_workspace_bytes) policy_loss_workspace_bytes = nullptr;
    decltype(&::wkv6_preference_loss) preference_loss = nullptr;
    decltype(&::wkv6_preference_loss_workspace_bytes) preference_loss_workspace_bytes = nullptr;
    decltype(&::wkv6_adamw_step) adamw_step = nullptr;
    decltype(&::wkv6_last_error) last_error = nullptr;
    bool bound = false;
} api;

void ok(int rc) { TORCH_CHECK(rc == 0, "wkv6_b200 error ", rc, ": ", api.last_error()); }

// Within a level of forward-mode differentiation any tensor may carry a tangent, which no call here carries on: the Python path looks at
// each.  (Here that would cost 20 ns a tensor, 4 us of the 12 that a step over 54 takes.)
bool ready() { return api.bound && plain_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr; }

Tensor floats(at::IntArrayRef sizes, const Tensor &like) {
    return at::detail::empty_cuda(sizes, at::kFloat, like.device(), std::nullopt);
}

float *ptr(const Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// What goes with the logits (a struct: only the logits are inputs of a node, and the mask may be undefined).
struct Given {
    Tensor targets, mask;
    double temperature;
};

// The rows of a call: logits [..., V] with one target, and maybe one mask byte, for each.
struct Rows {
    wkv6_token_logits p{};
    Tensor z, targets, mask;     // what p points into
    int64_t S = 1, T = 1;
};

// False where the call needs the Python path: other types, shapes that do not fit, layouts that need a copy of the logits, no rows.
bool describe(const Tensor &logits, const Given &given, Rows &r) {
    const auto &[targets, mask, temperature] = given;
    const int64_t d = logits.dim();
    if (d < 1 || targets.dim() != d - 1 || dtype_code(logits.scalar_type()) < 0 || targets.scalar_type() != at::kLong) return false;
    const int64_t V = logits.size(d - 1), rows = targets.numel();
    if (V < 1 || V > (1LL << 30) || rows < 1 || rows >= (1LL << 31)) return false;
    if (!std::equal(targets.sizes().begin(), targets.sizes().end(), logits.sizes().begin()) || targets.device() != logits.device()) return false;
    if (mask.defined() && (mask.scalar_type() != at::kBool || mask.sizes() != targets.sizes() || mask.device() != logits.device())) return false;
    if (V > 1 && logits.stride(d - 1) != 1) return false;
    r.T = d > 1 ? logits.size(d - 2) : 1;
    r.S = rows / r.T;
    if (d > 3 && !logits.is_contiguous()) return false;
    const int64_t row = r.T > 1 ? logits.stride(d - 2) : V, seq = r.S > 1 ? (d > 3 ? r.T * V : logits.stride(0)) : r.T * row;
    if (row <= 0 || seq <= 0) return false;
    r.z = logits;
    r.targets = targets.contiguous();
    if (mask.defined()) r.mask = mask.contiguous();
    r.p.S = (int32_t)r.S;
    r.p.T = (int32_t)r.T;
    r.p.V = (int32_t)V;
    r.p.dtype = dtype_code(logits.scalar_type());
    r.p.temperature = (float)temperature;
    if (!(r.p.temperature >= 1e-30f) || std::isinf(r.p.temperature)) return false;
    r.p.row_stride = row;
    r.p.seq_stride = seq;
    r.p.logits = logits.const_data_ptr();
    r.p.targets = r.targets.const_data_ptr<int64_t>();
    r.p.mask = mask.defined() ? static_cast<const uint8_t *>(r.mask.const_data_ptr()) : nullptr;
    return true;
}

// A gradient's factor or its values per token as dense fp32; an error where it is not a plain tensor (batched gradients).
Tensor dense_floats(Tensor g) {
    TORCH_CHECK_NOT_IMPLEMENTED(!g._fw_grad(0).defined(), "the backward of the losses has no forward-mode derivative");
    if (g.is_neg()) g = g.resolve_neg();
    TORCH_CHECK(plain_storage(g), "the backward of the losses takes plain tensors (no batched gradients)");
    return g.to(at::kFloat).contiguous();
}

Tensor empty_like_logits(const Tensor &logits) {
    return at::detail::empty_cuda(logits.sizes(), logits.scalar_type(), logits.device(), std::nullopt);
}

// Gradients as they leave a node: a derivative of the gradient is not available, and says so when it is asked for.
variable_list once(Tensor g, size_t inputs, const char *what) {
    variable_list out{g};
    if (at::GradMode::is_enabled()) {
        auto err = std::make_shared<torch::autograd::DelayedError>(what, 1);
        out[0] = out[0].detach().requires_grad_(true);
        out = (*err)(std::move(out));
    }
    out.resize(inputs);
    return out;
}

// One buffer holds what the backward of a loss needs of the rows: n coefficients, then the statistics at an 8-byte boundary.
float *stat_of(const Tensor &kept, int64_t n) { return ptr(kept) + (n + 1) / 2 * 2; }

void gradient(const Rows &r, const float *stat, const float *coefficient, bool per_sequence, const Tensor &factor, bool unless_one, Tensor &g) {
    ok(api.token_log_probs_backward(&r.p, stat, coefficient, per_sequence, ptr(factor), unless_one, g.data_ptr(), stream_of(g)));
}

Rows rows_again(const variable_list &saved, double temperature) {
    Rows r;
    TORCH_CHECK(describe(saved[0], {saved[1], saved[2], temperature}, r), "wkv6: unsupported call");     // checked by the forward
    return r;
}

// ------------------------------------------------------------------------------------------------------ log-probabilities

Tensor log_probs(const Rows &r, const Tensor &targets, Tensor *stat) {
    Tensor lp = floats(targets.sizes(), r.z);
    if (stat) *stat = floats({r.S * r.T, 2}, r.z);
    ok(api.token_log_probs(&r.p, ptr(lp), stat ? ptr(*stat) : nullptr, stream_of(lp)));
    return lp;
}

struct TokenLogProbs : public torch::autograd::Function<TokenLogProbs> {
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Given &given) {
        Rows r;
        TORCH_CHECK(describe(logits, given, r), "wkv6: unsupported call");        // checked by the caller
        Tensor stat, lp = log_probs(r, given.targets, &stat);
        ctx->save_for_backward({logits, r.targets, given.mask, stat});
        ctx->saved_data["temperature"] = given.temperature;
        return lp;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        Tensor g;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(s[0].device());
            const Rows r = rows_again(s, ctx->saved_data["temperature"].toDouble());
            g = empty_like_logits(s[0]);
            const Tensor coefficient = dense_floats(grads[0]);
            gradient(r, ptr(s[3]), ptr(coefficient), false, Tensor(), false, g);
        }
        return once(g, 2, "the gradient of token_log_probs is not differentiable");
    }
};

// ------------------------------------------------------------------------------------------------------------ policy loss

struct PolicyCall {
    Tensor advantages, old_lp, ref_lp;
    double low = 0, high = 0, kl = 0, scale = 1;
    int32_t reduction = 0;
};

// kept: what the backward needs of the rows (the coefficients [rows], the statistics [rows, 2]), and behind it the workspace
struct PolicyResult {
    Tensor loss, lp, kept, g;
};

PolicyResult policy(const Rows &r, const Tensor &targets, const PolicyCall &c, bool want_grad) {
    PolicyResult o;
    const int64_t rows = r.S * r.T, held = (rows * 3 + 1 + 3) / 4 * 4;      // the workspace at a 16-byte boundary
    const size_t nbytes = api.policy_loss_workspace_bytes(r.p.S, r.p.T, c.reduction);
    o.loss = floats({}, r.z);
    o.lp = floats(targets.sizes(), r.z);
    o.kept = floats({held + (int64_t)(nbytes + 3) / 4}, r.z);
    if (want_grad) o.g = empty_like_logits(r.z);
    float *coefficient = ptr(o.kept), *stat = stat_of(o.kept, rows);
    wkv6_policy q{};
    q.advantages = ptr(c.advantages);
    const int64_t d = c.advantages.dim();      // more than two: dense
    q.advantage_row_stride = d == 1 || d == 2 ? c.advantages.stride(d - 1) : 1;
    q.advantage_seq_stride = d == 2 ? c.advantages.stride(0) : r.T;
    q.old_log_probs = ptr(c.old_lp);
    q.ref_log_probs = ptr(c.ref_lp);
    q.clip_low = c.low;
    q.clip_high = c.high;
    q.kl_coef = c.kl;
    q.scale = c.scale;
    q.reduction = c.reduction;
    ok(api.policy_loss(&r.p, &q, ptr(o.loss), ptr(o.lp), stat, coefficient, want_grad ? o.g.data_ptr() : nullptr, ptr(o.kept) + held, nbytes,
                       stream_of(o.lp)));
    return o;
}

// The forward leaves the gradient for a loss that is the end of the graph; for another factor, a second backward, or one that is
// captured into a graph that the forward is not part of, it is formed anew from the logits (the first one belongs to whoever received
// it, and a replay must not find it as the last one left it).
struct PolicyLoss : public torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Given &given, const PolicyCall &c) {
        Rows r;
        TORCH_CHECK(describe(logits, given, r), "wkv6: unsupported call");
        PolicyResult o = policy(r, given.targets, c, true);
        ctx->save_for_backward({logits, r.targets, given.mask, o.kept});
        ctx->saved_data["temperature"] = given.temperature;
        ctx->saved_data["g"] = o.g;
        ctx->saved_data["capture"] = (int64_t)api.capture_id(stream_of(o.lp));
        ctx->mark_non_differentiable({o.lp});
        ctx->set_materialize_grads(false);
        return {o.loss, o.lp};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        if (!grads[0].defined()) return variable_list(3);
        Tensor g;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(s[0].device());
            const Rows r = rows_again(s, ctx->saved_data["temperature"].toDouble());
            const Tensor factor = dense_floats(grads[0]);
            auto kept = ctx->saved_data.find("g");
            bool first = kept != ctx->saved_data.end();
            if (first) {
                g = kept->second.toTensor();
                ctx->saved_data.erase(kept);
                first = (int64_t)api.capture_id(stream_of(g)) == ctx->saved_data["capture"].toInt();
            }
            if (!first) g = empty_like_logits(s[0]);
            gradient(r, stat_of(s[3], r.S * r.T), ptr(s[3]), false, factor, first, g);
        }
        return once(g, 3, "the gradient of policy_loss is not differentiable");
    }
};

// -------------------------------------------------------------------------------------------------------- preference loss

struct PreferenceCall {
    Tensor ref;
    double beta = 0, smoothing = 0, margin = 0, scale = 1;
    bool average = false;
};

// kept: the coefficients [S] and statistics [rows, 2], and behind them the rows' log-probabilities and the workspace
struct PreferenceResult {
    Tensor loss, seq, kept;
};

PreferenceResult preference(const Rows &r, const PreferenceCall &c, bool want_grad) {
    PreferenceResult o;
    const int64_t rows = r.S * r.T, held = (r.S + 1) / 2 * 2 + rows * 2, more = held + (rows + 1) / 2 * 2;      // even: 8-byte boundaries
    const size_t nbytes = api.preference_loss_workspace_bytes(r.p.S);
    o.loss = floats({}, r.z);
    o.seq = floats({r.S}, r.z);
    o.kept = floats({more + (int64_t)(nbytes + 3) / 4}, r.z);
    float *coefficient = ptr(o.kept), *lp = coefficient + held;
    void *stream = stream_of(o.seq);
    ok(api.token_log_probs(&r.p, lp, want_grad ? stat_of(o.kept, r.S) : nullptr, stream));
    wkv6_preference q{};
    q.ref_log_probs = ptr(c.ref);
    q.beta = c.beta;
    q.label_smoothing = c.smoothing;
    q.margin = c.margin;
    q.scale = c.scale;
    q.average = c.average;
    ok(api.preference_loss(&r.p, lp, &q, ptr(o.loss), ptr(o.seq), coefficient, coefficient + more, nbytes, stream));
    return o;
}

struct PreferenceLoss : public torch::autograd::Function<PreferenceLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Given &given, const PreferenceCall &c) {
        Rows r;
        TORCH_CHECK(describe(logits, given, r), "wkv6: unsupported call");
        PreferenceResult o = preference(r, c, true);
        ctx->save_for_backward({logits, r.targets, given.mask, o.kept});
        ctx->mark_non_differentiable({o.seq});
        ctx->set_materialize_grads(false);
        return {o.loss, o.seq};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        if (!grads[0].defined()) return variable_list(3);
        Tensor g;
        {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(s[0].device());
            const Rows r = rows_again(s, 1.0);
            g = empty_like_logits(s[0]);
            gradient(r, stat_of(s[3], r.S), ptr(s[3]), true, dense_floats(grads[0]), false, g);
        }
        return once(g, 3, "the gradient of preference_loss is not differentiable");
    }
};

// -------------------------------------------------------------------------------------------------------- from Python

// args[i] as a plain tensor; None as an undefined one where it may be left out
bool tensor_arg(PyObject *o, Tensor &t, bool optional) {
    if (optional && o == Py_None) return true;
    if (!plain_tensor(o)) return false;
    t = THPVariable_Unpack(o);
    return true;
}

// A constant of the loss: fp32, of these sizes; dense, or (strided) with strides for the sequence and the token
bool constant_arg(PyObject *o, Tensor &t, at::IntArrayRef sizes, const Tensor &logits, bool optional, bool strided = false) {
    if (!tensor_arg(o, t, optional)) return false;
    if (!t.defined()) return true;
    if (!at::isFloatingType(t.scalar_type()) || t.sizes() != sizes || t.device() != logits.device()) return false;
    if (t.requires_grad()) {
        if (at::GradMode::is_enabled()) return false;
        t = t.detach();
    }
    if (t.scalar_type() != at::kFloat) t = t.to(at::kFloat);
    if (!t.is_contiguous() && !(strided && t.dim() <= 2)) t = t.contiguous();
    return true;
}

bool needs_grad(const Tensor &logits) { return at::GradMode::is_enabled() && logits.requires_grad(); }

PyObject *pair(Tensor a, Tensor b) {
    PyObject *t = PyTuple_New(2);
    if (t == nullptr) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
    return t;
}

bool numbers(PyObject *const *args, int n, double *out) {
    for (int i = 0; i < n; ++i) {
        if (!PyFloat_Check(args[i]) && !PyLong_Check(args[i])) return false;
        out[i] = PyFloat_AsDouble(args[i]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return false;
        }
    }
    return true;
}

}  // namespace

// token_log_probs(logits, targets, mask or None, temperature) -> lp or None
PyObject *py_token_log_probs(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor logits, lp;
    Given given;
    Rows r;
    if (n != 4 || !ready() || !tensor_arg(args[0], logits, false) || !tensor_arg(args[1], given.targets, false) || !tensor_arg(args[2], given.mask, true) ||
        !numbers(args + 3, 1, &given.temperature) || !describe(logits, given, r))
        return none();
    {
        pybind11::gil_scoped_release no_gil;
        c10::cuda::CUDAGuard guard(logits.device());
        lp = needs_grad(logits) ? TokenLogProbs::apply(logits, given) : log_probs(r, given.targets, nullptr);
    }
    return THPVariable_Wrap(std::move(lp));
    END_HANDLE_TH_ERRORS
}

// policy_loss(logits, targets, mask or None, advantages, old, ref or None, temperature, clip_low, clip_high, kl_coef, scale, reduction)
// -> (loss, lp) or None
PyObject *py_policy_loss(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor logits;
    Given given;
    PolicyCall c;
    double x[5];
    Rows r;
    if (n != 12 || !ready() || !tensor_arg(args[0], logits, false) || !tensor_arg(args[1], given.targets, false) || !tensor_arg(args[2], given.mask, true) ||
        !numbers(args + 6, 5, x) || !PyLong_Check(args[11]))
        return none();
    given.temperature = x[0];
    if (!describe(logits, given, r)) return none();
    if (!constant_arg(args[3], c.advantages, given.targets.sizes(), logits, false, true) || !constant_arg(args[4], c.old_lp, given.targets.sizes(), logits, false) ||
        !constant_arg(args[5], c.ref_lp, given.targets.sizes(), logits, true))
        return none();
    c.low = x[1];
    c.high = x[2];
    c.kl = x[3];
    c.scale = x[4];
    c.reduction = (int32_t)PyLong_AsLong(args[11]);
    Tensor loss, lp;
    {
        pybind11::gil_scoped_release no_gil;
        c10::cuda::CUDAGuard guard(logits.device());
        if (needs_grad(logits)) {
            variable_list out = PolicyLoss::apply(logits, given, c);
            loss = out[0];
            lp = out[1];
        } else {
            PolicyResult o = policy(r, given.targets, c, false);
            loss = o.loss;
            lp = o.lp;
        }
    }
    return pair(std::move(loss), std::move(lp));
    END_HANDLE_TH_ERRORS
}

// preference_loss(logits, targets, mask or None, ref or None, beta, label_smoothing, margin, scale, average) -> (loss, seq) or None
PyObject *py_preference_loss(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor logits;
    Given given;
    PreferenceCall c;
    double x[4];
    Rows r;
    if (n != 9 || !ready() || !tensor_arg(args[0], logits, false) || !tensor_arg(args[1], given.targets, false) || !tensor_arg(args[2], given.mask, true) ||
        !numbers(args + 4, 4, x) || given.targets.dim() != 2 || given.targets.size(0) % 2)
        return none();
    given.temperature = 1.0;
    if (!describe(logits, given, r)) return none();
    if (!constant_arg(args[3], c.ref, {given.targets.size(0)}, logits, true)) return none();
    c.beta = x[0];
    c.smoothing = x[1];
    c.margin = x[2];
    c.scale = x[3];
    c.average = args[8] == Py_True;
    Tensor loss, seq;
    {
        pybind11::gil_scoped_release no_gil;
        c10::cuda::CUDAGuard guard(logits.device());
        if (needs_grad(logits)) {
            variable_list out = PreferenceLoss::apply(logits, given, c);
            loss = out[0];
            seq = out[1];
        } else {
            PreferenceResult o = preference(r, c, false);
            loss = o.loss;
            seq = o.seq;
        }
    }
    return pair(std::move(loss), std::move(seq));
    END_HANDLE_TH_ERRORS
}

namespace {

struct Span {
    uintptr_t begin, end;
    bool operator<(const Span &o) const { return begin < o.begin; }
};

// The tensors of a list, which stay where the list holds them; false where one is not plain, dense, of this type or on this device.
bool list_arg(PyObject *list, Py_ssize_t count, c10::Device dev, std::vector<const Tensor *> &out) {
    if (!PyList_CheckExact(list) || PyList_GET_SIZE(list) != count) return false;
    out.resize(count);
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject *o = PyList_GET_ITEM(list, i);
        if (!plain_tensor(o)) return false;
        const Tensor &t = THPVariable_Unpack(o);
        if (t.device() != dev || !t.is_contiguous()) return false;
        out[i] = &t;
    }
    return true;
}

// Adds a list's spans to the sorted ones.  Tensors of a model mostly lie in the order in which they were made, so that there is
// little to sort.
void add_spans(const std::vector<const Tensor *> &ts, std::vector<Span> &spans) {
    const size_t old = spans.size();
    for (const Tensor *t : ts)
        if (const size_t nbytes = t->nbytes()) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(t->const_data_ptr());
            spans.push_back({a, a + nbytes});
        }
    if (!std::is_sorted(spans.begin() + old, spans.end())) std::sort(spans.begin() + old, spans.end());
    std::inplace_merge(spans.begin(), spans.begin() + old, spans.end());
}

// A number, or one value of `type` on the device
bool value_arg(PyObject *o, at::ScalarType type, c10::Device dev, const void **device) {
    if (!plain_tensor(o)) return false;
    const Tensor &t = THPVariable_Unpack(o);
    if (t.scalar_type() != type || t.numel() != 1 || t.device() != dev) return false;
    *device = t.const_data_ptr();
    return true;
}

}  // namespace

// adamw_step(params, grads, exp_avgs, exp_avg_sqs, m_scales or None, v_scales or None, step, lr, beta1, beta2, eps, weight_decay, seed,
//            stochastic, grad_scale or None, first_index) -> True or None
PyObject *py_adamw_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 16 || !ready() || !PyList_CheckExact(args[0]) || PyList_GET_SIZE(args[0]) == 0 || (args[4] == Py_None) != (args[5] == Py_None))
        return none();
    if (!plain_tensor(PyList_GET_ITEM(args[0], 0))) return none();
    const c10::Device dev = THPVariable_Unpack(PyList_GET_ITEM(args[0], 0)).device();
    const Py_ssize_t count = PyList_GET_SIZE(args[0]);
    const bool narrow = args[4] != Py_None;
    std::vector<const Tensor *> lists[6];
    for (int k = 0; k < (narrow ? 6 : 4); ++k)
        if (!list_arg(args[k], count, dev, lists[k])) return none();
    const auto &p = lists[0], &g = lists[1], &m = lists[2], &v = lists[3], &ms = lists[4], &vs = lists[5];
    const at::ScalarType state = narrow ? at::kFloat8_e4m3fn : at::kFloat;
    wkv6_adamw c{};
    double x[4];
    if (!numbers(args + 8, 4, x) || !(x[0] >= 0.0 && x[0] < 1.0 && x[1] >= 0.0 && x[1] < 1.0) || !(x[2] == 0.0 || (x[2] >= FLT_MIN && x[2] <= FLT_MAX)) || !std::isfinite(x[3]))
        return none();
    c.state_bits = narrow ? 8 : 32;
    if (narrow && x[0] > 0.94) return none();
    c.beta1 = x[0];
    c.beta2 = x[1];
    c.eps = x[2];
    c.weight_decay = x[3];
    const void *at_device = nullptr;
    if (PyLong_CheckExact(args[6])) {
        c.step = PyLong_AsLongLong(args[6]);
        if (PyErr_Occurred()) PyErr_Clear();       // -1
        if (c.step < 1) return none();
    } else {
        if (!value_arg(args[6], at::kLong, dev, &at_device)) return none();
        c.step_device = static_cast<const int64_t *>(at_device);
    }
    if (numbers(args + 7, 1, &c.lr)) {
        if (!std::isfinite(c.lr)) return none();
    } else {
        if (!value_arg(args[7], at::kFloat, dev, &at_device)) return none();
        c.lr_device = static_cast<const float *>(at_device);
    }
    if (!PyLong_CheckExact(args[12]) || !PyLong_CheckExact(args[15])) return none();
    const unsigned long long seed = PyLong_AsUnsignedLongLongMask(args[12]);
    const long long first = PyLong_AsLongLong(args[15]);
    if (PyErr_Occurred()) PyErr_Clear();           // -1
    if (first < 0 || first + count > 0x7fffffffLL) return none();
    c.seed = (int64_t)seed;
    c.stochastic = args[13] == Py_True;
    if (args[14] != Py_None) {
        if (!value_arg(args[14], at::kFloat, dev, &at_device)) return none();
        c.grad_scale = static_cast<const float *>(at_device);
    }
    std::vector<wkv6_adamw_tensor> table[2];       // bf16, fp32
    for (auto &x : table) x.reserve(count);
    for (Py_ssize_t i = 0; i < count; ++i) {
        const int64_t size = p[i]->numel(), blocks = (size + 255) / 256;
        const at::ScalarType t = p[i]->scalar_type();
        if ((t != at::kBFloat16 && t != at::kFloat) || g[i]->scalar_type() != t || m[i]->scalar_type() != state || v[i]->scalar_type() != state ||
            g[i]->numel() != size || m[i]->numel() != size || v[i]->numel() != size || p[i]->is_inference())
            return none();
        wkv6_adamw_tensor e{};
        if (narrow) {
            if (ms[i]->scalar_type() != at::kFloat || vs[i]->scalar_type() != at::kFloat || ms[i]->numel() != blocks || vs[i]->numel() != blocks) return none();
            e.m_scale = static_cast<float *>(ms[i]->data_ptr());
            e.v_scale = static_cast<float *>(vs[i]->data_ptr());
        }
        e.p = p[i]->data_ptr();
        e.g = g[i]->const_data_ptr();
        e.m = m[i]->data_ptr();
        e.v = v[i]->data_ptr();
        e.n = size;
        e.index = first + i;
        table[t == at::kFloat].push_back(e);
    }
    std::vector<Span> spans;
    spans.reserve(count * (narrow ? 5 : 3));
    for (int k : {0, 2, 3, 4, 5})
        if (!lists[k].empty()) add_spans(lists[k], spans);
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i].begin < spans[i - 1].end) return none();
    for (const Tensor *t : g) {      // gradients may share memory among themselves only
        const uintptr_t a = reinterpret_cast<uintptr_t>(t->const_data_ptr()), b = a + t->nbytes();
        const auto next = std::lower_bound(spans.begin(), spans.end(), Span{b, b});      // the first that begins at or behind its end
        if (a < b && next != spans.begin() && (next - 1)->end > a) return none();
    }
    {
        c10::cuda::CUDAGuard guard(dev);
        if (c.step_device == nullptr && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return none();
        for (int k = 0; k < 2; ++k) {
            if (table[k].empty()) continue;
            c.dtype = k ? WKV6_F32 : WKV6_BF16;
            ok(api.adamw_step(&c, (int64_t)table[k].size(), table[k].data(), stream_of(*p[0])));
        }
    }
    for (int k : {0, 2, 3, 4, 5})
        for (const Tensor *t : lists[k])
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

const char *bind_training(void *library) {
#define SYM(name)                                                                                                                  \
    if ((api.name = reinterpret_cast<decltype(api.name)>(dlsym(library, "wkv6_" #name))) == nullptr) return "wkv6_" #name;
    SYM(token_log_probs) SYM(token_log_probs_backward) SYM(capture_id) SYM(policy_loss) SYM(policy_loss_workspace_bytes) SYM(preference_loss)
    SYM(preference_loss_workspace_bytes) SYM(adamw_step) SYM(last_error)
#undef SYM
    api.bound = true;
    return nullptr;
}

}  // namespace wkv6_native
