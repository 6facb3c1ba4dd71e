// The trainer-side operators as torch sees them (mpe_hip/learn.py): argument checks, output buffers, the current stream, and
// the autograd nodes, in C++ so that neither the calls nor the backward pass, which torch runs on a thread of its own, wait
// for the interpreter.  The work itself is behind the C ABI: bind() hands over the addresses of the library that
// mpe_hip/_lib.py has loaded, so there is one library in the process whichever build it is.
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/mpe_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

namespace {

struct Api {
    decltype(&mpe_last_error) last_error;
    decltype(&mpe_linear_workspace) linear_workspace;
    decltype(&mpe_linear_forward) linear_forward;
    decltype(&mpe_linear_backward) linear_backward;
    decltype(&mpe_ppo_loss_forward) ppo_forward;
    decltype(&mpe_ppo_loss_backward) ppo_backward;
    decltype(&mpe_clip_grad_norm) clip;
} api;

struct Failure : std::runtime_error {       // becomes MpeError where Python is the caller
    int code;
    Failure(int c, const char* what) : std::runtime_error(what), code(c) {}
};

void check(int rc) {
    if (rc == MPE_OK) return;
    const char* what = api.last_error(nullptr);
    throw Failure(rc, what ? what : "?");
}

constexpr int64_t ROW_MAX = (int64_t)1 << 22;      // the longest row stride the kernels take

int type_code(at::ScalarType t) {
    return t == at::kFloat ? MPE_F32 : t == at::kBFloat16 ? MPE_BF16 : t == at::kHalf ? MPE_F16 : -1;
}

int type_of(const Tensor& t, const char* who) {
    TORCH_CHECK_VALUE(t.is_cuda(), who, " needs GPU tensors; there is no CPU path");
    const int code = type_code(t.scalar_type());
    TORCH_CHECK_VALUE(code >= 0 && t.layout() == at::kStrided, who, " takes dense float32, bfloat16 or float16, not ", t.scalar_type());
    return code;
}

bool has(const MaybeTensor& t) { return t.has_value() && t->defined(); }

// A forward-mode tangent would be lost without a word: a result without one counts as constant.
void no_tangent(const MaybeTensor& t, const char* who) {
    TORCH_CHECK_NOT_IMPLEMENTED(!has(t) || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t->_fw_grad(0).defined(), who,
                                ": forward-mode derivatives are not available");
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
mpe_stream_t stream_of(const Tensor& t) { return (mpe_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor bytes_like(int64_t n, const Tensor& t) { return n > 0 ? at::empty({n}, t.options().dtype(at::kByte)) : Tensor(); }

// A tensor as rows of `cols` contiguous elements, any row stride >= cols; copied only if it has to be.
struct Rows {
    Tensor t;
    int64_t ld;
};

Rows rows_of(const Tensor& t, int64_t cols) {
    if (t.is_neg()) return rows_of(t.resolve_neg(), cols);      // memory that holds the negative of its numbers
    if (t.is_contiguous()) return {t, cols};
    Tensor m = t.dim() == 2 ? t : t.reshape({-1, cols});
    const int64_t rows = m.size(0), ld = m.stride(0);
    if ((cols > 1 && m.stride(1) != 1) || (rows > 1 && (ld < cols || ld > ROW_MAX))) return {m.contiguous(), cols};
    return {m, rows > 1 ? ld : cols};       // a single row's stride says nothing
}

// One row of a vector's length or more that expand() repeats stays one row: stride 0.
Rows rows_or_one(const Tensor& t, int64_t cols) {
    if (cols >= 8 && !t.is_neg() && !t.is_contiguous() && t.dim() >= 2 && t.numel() > 0 && t.stride(-1) == 1) {
        bool one = true;
        for (int64_t d = 0; d + 1 < t.dim(); ++d) one = one && (t.stride(d) == 0 || t.size(d) == 1);
        if (one) return {t, 0};
    }
    return rows_of(t, cols);
}

// t itself, or its copy if rows_of had to make one
Tensor as_taken(const Tensor& t, const Rows& rows) { return rows.t.is_alias_of(t) ? t : rows.t.view(t.sizes()); }

Tensor flat(const Tensor& t) { return t.defined() && (!t.is_contiguous() || t.is_neg()) ? t.resolve_neg().contiguous() : t; }

// Gradients that cannot be differentiated again say so if it is tried.
variable_list once(variable_list grads, const char* who) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in, out(grads.size());
    for (auto& g : grads)
        if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
    if (in.empty()) return grads;
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(who) + ": second derivatives are not available", (int)in.size());
    variable_list got = (*node)(std::move(in));
    size_t k = 0;
    for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) out[i] = got[k++];
    return out;
}

// ---- linear ----

Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int act, int code, bool keep, Tensor* pre) {
    const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
    const Rows x2 = rows_of(x, k), w2 = rows_of(w, k);
    const Rows r2 = r.defined() ? rows_or_one(r, n) : Rows{Tensor(), 0};
    const Tensor b1 = flat(b);
    auto shape = x.sizes().vec();
    shape.back() = n;
    Tensor y = at::empty(shape, x.options());
    if (keep) *pre = at::empty({m, n}, act == MPE_ACT_RELU ? x.options() : x.options().dtype(code == MPE_BF16 ? at::kHalf : at::kFloat));
    int64_t need = 0;
    check(api.linear_workspace(code, act, m, n, k, &need, nullptr));
    const Tensor ws = bytes_like(need, x);
    check(api.linear_forward(x.device().index(), code, act, m, n, k, ptr(x2.t), x2.ld, ptr(w2.t), w2.ld, ptr(b1), ptr(r2.t), r2.ld, ptr(y), n,
                             keep ? ptr(*pre) : nullptr, ptr(ws), need, stream_of(x)));
    return y;
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const MaybeTensor& b, const MaybeTensor& r, int64_t act, int64_t code) {
        // where nothing was added to it, the output itself tells relu's slope, and in float32 tanh's
        const bool from_y = !has(r) && (act == MPE_ACT_RELU || (act == MPE_ACT_TANH && code == MPE_F32));
        const bool keep = act != MPE_ACT_NONE && !from_y;
        Tensor pre;
        Tensor y = linear_forward(x, w, has(b) ? *b : Tensor(), has(r) ? *r : Tensor(), (int)act, (int)code, keep, &pre);
        ctx->saved_data["a"] = (int64_t)(from_y && act == MPE_ACT_TANH ? MPE_ACT_TANH_OUT : act) | (has(b) ? 16 : 0) | (has(r) ? 32 : 0) | code << 8;
        ctx->save_for_backward({x, w, keep ? pre : act != MPE_ACT_NONE ? y : Tensor()});
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const int64_t a = ctx->saved_data["a"].toInt();
        const int act = a & 15, code = (int)(a >> 8);
        const bool with_b = a & 16, with_r = a & 32;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &pre = saved[2], &dy = grads[0];
        if (!dy.defined()) return variable_list(6);
        no_tangent(dy, "linear");
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool need_b = with_b && ctx->needs_input_grad(2), need_r = with_r && ctx->needs_input_grad(with_b ? 3 : 2);
        Tensor dx, dw, db;
        if (need_x || need_w || need_b) {
            const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
            const Rows x2 = rows_of(x, k), w2 = rows_of(w, k), d2 = rows_or_one(dy, n);
            if (need_x) dx = at::empty(x.sizes(), x.options());
            if (need_w) dw = at::empty({n, k}, x.options());
            if (need_b) db = at::empty({n}, x.options());
            int64_t need = 0;
            check(api.linear_workspace(code, act, m, n, k, nullptr, &need));
            const Tensor ws = bytes_like(need, x);
            check(api.linear_backward(x.device().index(), code, act, m, n, k, ptr(d2.t), d2.ld, ptr(x2.t), x2.ld, ptr(w2.t), w2.ld, ptr(pre), ptr(dx), k, ptr(dw),
                                      ptr(db), ptr(ws), need, stream_of(x)));
        }
        return once({dx, dw, db, need_r ? dy : Tensor(), Tensor(), Tensor()}, "linear");
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const MaybeTensor& b, const MaybeTensor& r, int64_t act) {
    for (const MaybeTensor& t : {MaybeTensor(x), MaybeTensor(w), b, r}) no_tangent(t, "linear");
    const int code = type_of(x, "linear");
    TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.size(0) >= 1 && w.size(1) >= 1,
                      "linear: x [..., k] and weight [n, k], n and k at least 1; got ", x.sizes(), " and ", w.sizes());
    const int64_t n = w.size(0);
    bool needs = x.requires_grad() || w.requires_grad();
    const auto same = [&](const Tensor& t, const char* name) {
        TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.layout() == at::kStrided, "linear: ", name,
                          " must share x's type and device (", x.scalar_type(), ", ", x.device(), ")");
        needs = needs || t.requires_grad();
    };
    same(w, "weight");
    if (has(b)) {
        TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == n, "linear: bias must have shape (", n, ",), got ", b->sizes());
        same(*b, "bias");
    }
    if (has(r)) {
        bool ok = r->dim() == x.dim() && r->size(-1) == n;
        for (int64_t d = 0; ok && d + 1 < x.dim(); ++d) ok = r->size(d) == x.size(d);
        TORCH_CHECK_VALUE(ok, "linear: residual must have the result's shape, x's with ", n, " at the end, got ", r->sizes());
        same(*r, "residual");
    }
    if (needs && at::GradMode::is_enabled()) return Linear::apply(x, w, b, r, act, (int64_t)code);
    return linear_forward(x, w, has(b) ? *b : Tensor(), has(r) ? *r : Tensor(), (int)act, code, false, nullptr);
}

// ---- ppo_loss ----

struct PpoCoefs {
    double clip, value_clip, value_coef, entropy_coef;
};

struct PpoLoss : torch::autograd::Function<PpoLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const MaybeTensor& values, const std::vector<Tensor>* side, const PpoCoefs* q,
                                 int64_t code) {
        // side: actions, old_logp, adv, old_values, returns, mask, weights; the mask as rows, the others contiguous
        const int64_t v = logits.size(-1);
        const Rows l2 = rows_of(logits, v), m2 = (*side)[5].defined() ? rows_of((*side)[5], v) : Rows{Tensor(), 0};
        const Tensor val = has(values) ? flat(*values) : Tensor();
        const auto f32 = logits.options().dtype(at::kFloat);
        Tensor loss = at::empty({}, f32), stats = at::empty({6}, f32);
        const Tensor ws = bytes_like(MPE_PPO_WORKSPACE_BYTES, logits);
        const auto& s = *side;
        check(api.ppo_forward(logits.device().index(), (int)code, logits.numel() / v, v, ptr(l2.t), l2.ld, ptr(s[0]), (int)s[0].element_size(),
                              (const float*)ptr(s[1]), (const float*)ptr(s[2]), (const uint8_t*)ptr(m2.t), m2.ld, (const float*)ptr(s[6]), (const float*)ptr(val),
                              (const float*)ptr(s[3]), (const float*)ptr(s[4]), q->clip, q->value_clip, q->value_coef, q->entropy_coef, (float*)ptr(loss),
                              (float*)ptr(stats), ptr(ws), MPE_PPO_WORKSPACE_BYTES, stream_of(logits)));
        ctx->saved_data["a"] = code | (has(values) ? 16 : 0);
        ctx->saved_data["q"] = std::vector<double>{q->clip, q->value_clip, q->value_coef, q->entropy_coef};
        // what had to be copied is saved as it was copied
        ctx->save_for_backward({as_taken(logits, l2), val, stats, s[0], s[1], s[2], s[3], s[4], s[5], s[6]});
        ctx->mark_non_differentiable({stats});
        return {loss, stats};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined()) return variable_list(5);
        no_tangent(grads[0], "ppo_loss");
        const int64_t a = ctx->saved_data["a"].toInt();
        const auto q = ctx->saved_data["q"].toDoubleVector();
        const auto s = ctx->get_saved_variables();      // throws where an input was written since
        const Tensor &logits = s[0], &values = s[1];
        const bool need_l = ctx->needs_input_grad(0), need_v = (a & 16) && ctx->needs_input_grad(1);
        Tensor dl, dv;
        if (need_l || need_v) {
            const int64_t v = logits.size(-1);
            const Rows l2 = rows_of(logits, v), m2 = s[8].defined() ? rows_of(s[8], v) : Rows{Tensor(), 0};
            const Tensor grad = (grads[0].scalar_type() == at::kFloat ? grads[0] : grads[0].to(at::kFloat)).resolve_neg();
            if (need_l) dl = at::empty(logits.sizes(), logits.options());
            if (need_v) dv = at::empty(values.sizes(), values.options());
            check(api.ppo_backward(logits.device().index(), (int)(a & 15), logits.numel() / v, v, ptr(l2.t), l2.ld, ptr(s[3]), (int)s[3].element_size(),
                                   (const float*)ptr(s[4]), (const float*)ptr(s[5]), (const uint8_t*)ptr(m2.t), m2.ld, (const float*)ptr(s[9]),
                                   (const float*)ptr(values), (const float*)ptr(s[6]), (const float*)ptr(s[7]), q[0], q[1], q[2], q[3], (const float*)ptr(s[2]),
                                   (const float*)ptr(grad), ptr(dl), need_l ? v : 0, (float*)ptr(dv), stream_of(logits)));
        }
        return once({dl, dv, Tensor(), Tensor(), Tensor()}, "ppo_loss");
    }
};

py::tuple ppo_loss(const Tensor& logits, const Tensor& actions, const Tensor& old_logp, const Tensor& adv, const MaybeTensor& values, const MaybeTensor& old_values,
                   const MaybeTensor& returns, const MaybeTensor& mask, const MaybeTensor& weights, double clip, std::optional<double> value_clip, double value_coef,
                   double entropy_coef) {
    for (const MaybeTensor& t : {MaybeTensor(logits), MaybeTensor(old_logp), MaybeTensor(adv), values, old_values, returns, weights}) no_tangent(t, "ppo_loss");
    const int code = type_of(logits, "ppo_loss");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "ppo_loss: logits must be [..., v] with v at least 1, got ", logits.sizes());
    TORCH_CHECK_VALUE(has(values) == has(old_values) && has(values) == has(returns), "ppo_loss: values, old_values and returns go together");
    TORCH_CHECK_VALUE(actions.scalar_type() == at::kInt || actions.scalar_type() == at::kLong, "ppo_loss: actions must be int32 or int64, not ", actions.scalar_type());
    TORCH_CHECK_VALUE(clip >= 0 && (!value_clip || *value_clip >= 0), "ppo_loss: clip and value_clip must not be negative");
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    const auto side = [&](const char* name, const MaybeTensor& t, at::ScalarType type, at::IntArrayRef shape) {
        if (!has(t)) return Tensor();
        TORCH_CHECK_VALUE(t->scalar_type() == type, "ppo_loss: ", name, " must be ", type, ", not ", t->scalar_type());
        TORCH_CHECK_VALUE(t->sizes() == shape && t->device() == logits.device() && t->layout() == at::kStrided, "ppo_loss: ", name, " must have shape ", shape, " on ",
                          logits.device(), ", got ", t->sizes(), " on ", t->device());
        return *t;
    };
    Tensor m, w;
    if (has(mask)) {
        TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte, "ppo_loss: action_mask must be bool or uint8, not ", mask->scalar_type());
        m = side("action_mask", mask, mask->scalar_type(), logits.sizes());
        m = as_taken(m, rows_of(m, logits.size(-1)));
    }
    if (has(weights)) w = side("weights", weights->scalar_type() == at::kBool ? MaybeTensor(weights->to(at::kFloat)) : weights, at::kFloat, lead);
    side("values", values, at::kFloat, lead);
    const std::vector<Tensor> s = {flat(side("actions", actions, actions.scalar_type(), lead)), flat(side("old_logp", old_logp, at::kFloat, lead)),
                                   flat(side("advantages", adv, at::kFloat, lead)), flat(side("old_values", old_values, at::kFloat, lead)),
                                   flat(side("returns", returns, at::kFloat, lead)), m, flat(w)};
    const PpoCoefs q = {clip, value_clip.value_or(-1.0), value_coef, entropy_coef};
    const auto out = PpoLoss::apply(logits, values, &s, &q, (int64_t)code);
    return py::make_tuple(out[0], out[1].slice(0, 0, 5));
}

// ---- global norm ----

// t's elements fill one run of memory, in whatever order of dimensions
bool dense(const Tensor& t) { return !t.is_neg() && t.layout() == at::kStrided && (t.is_contiguous() || t.is_non_overlapping_and_dense()); }

Tensor clip(const std::vector<Tensor>& ts, double max_norm, const std::optional<std::vector<Tensor>>& outs) {
    const size_t n = ts.size();
    for (const Tensor& t : ts) no_tangent(t, "clip_grad_norm");
    if (outs)
        for (const Tensor& t : *outs) no_tangent(t, "clip_grad_norm");
    TORCH_CHECK_VALUE(n > 0, "clip_grad_norm: no tensors");
    TORCH_CHECK_VALUE(n <= 0x7fffffff, "clip_grad_norm: too many tensors");
    TORCH_CHECK_VALUE(max_norm >= 0, "clip_grad_norm: max_norm must not be negative, got ", max_norm);
    TORCH_CHECK_VALUE(!outs || outs->size() == n, "clip_grad_norm: ", n, " tensors but ", outs ? outs->size() : 0, " in out");
    const auto dev = ts[0].device();
    std::vector<const void*> src(n);
    std::vector<void*> dst(outs ? n : 0);
    std::vector<int64_t> count(n);
    std::vector<int32_t> type(n);
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (size_t i = 0; i < n; ++i) {
        const Tensor& t = ts[i];
        type[i] = type_code(t.scalar_type());
        TORCH_CHECK_VALUE(t.is_cuda() && t.device() == dev && type[i] >= 0, "clip_grad_norm: tensor ", i,
                          " must be float32, bfloat16 or float16 on the GPU of tensor 0 (", dev, "), got ", t.scalar_type(), " on ", t.device());
        TORCH_CHECK_VALUE(dense(t), "clip_grad_norm: tensor ", i, " is sparse, a negative view or has gaps or repeated elements");
        src[i] = t.data_ptr();
        count[i] = t.numel();
        if (!outs) continue;
        const Tensor& o = (*outs)[i];
        TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !o.requires_grad(), "clip_grad_norm: out ", i, " requires gradients, which clipping does not have");
        if (!o.is_same(t))
            TORCH_CHECK_VALUE(!o.is_neg() && o.layout() == at::kStrided && o.scalar_type() == t.scalar_type() && o.device() == dev && o.sizes() == t.sizes() &&
                                  ((o.is_contiguous() && t.is_contiguous()) || o.strides() == t.strides()),
                              "clip_grad_norm: out ", i, " must have the shape, strides, type and device of its tensor");
        dst[i] = o.data_ptr();
        if (count[i]) spans.push_back({(uintptr_t)dst[i], (uintptr_t)dst[i] + (uintptr_t)count[i] * o.element_size()});
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second, "clip_grad_norm: a tensor is given twice, or two share memory");
    Tensor norm = at::empty({}, ts[0].options().dtype(at::kFloat).requires_grad(false));
    const Tensor ws = bytes_like(MPE_CLIP_WORKSPACE_BYTES, norm);
    check(api.clip(dev.index(), (int32_t)n, src.data(), outs ? dst.data() : nullptr, count.data(), type.data(), max_norm, (float*)ptr(norm), ptr(ws),
                   MPE_CLIP_WORKSPACE_BYTES, stream_of(norm)));
    if (outs)
        for (const Tensor& o : *outs)
            if (!o.is_inference()) torch::autograd::impl::bump_version(o);
    return norm;
}

template <typename F>
void take(const py::dict& d, const char* name, F& f) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }

}  // namespace

PYBIND11_MODULE(_native, m) {
    static py::handle error;        // lives as long as the process
    m.def("bind", [](const py::dict& d, py::object mpe_error) {
        take(d, "mpe_last_error", api.last_error);
        take(d, "mpe_linear_workspace", api.linear_workspace);
        take(d, "mpe_linear_forward", api.linear_forward);
        take(d, "mpe_linear_backward", api.linear_backward);
        take(d, "mpe_ppo_loss_forward", api.ppo_forward);
        take(d, "mpe_ppo_loss_backward", api.ppo_backward);
        take(d, "mpe_clip_grad_norm", api.clip);
        error = mpe_error.release();
    });
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& f) {
            py::object e = py::reinterpret_borrow<py::object>(error)(f.code, f.what());
            PyErr_SetObject(error.ptr(), e.ptr());
        }
    });
    m.def("linear", &linear);
    m.def("ppo_loss", &ppo_loss);
    m.def("clip", &clip);
}
