// sb_torch.cpp -- the policy operators as torch operators with gradients.
//
// A call's arguments are checked, its outputs allocated and its kernel launched
// here, and the gradient is a node of autograd's own kind: for a small batch
// the host's work is the whole cost (a training call of 64 rows took 99 us
// through a Python autograd function, of which 50 are autograd's engine).
// The kernels stay behind the C ABI: bind() receives the addresses of its
// entry points, so this file links against torch alone.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <vector>

#include "stratego_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
    decltype(&sb_action_logprobs) logprobs = nullptr;
    decltype(&sb_action_logprobs_backward) logprobs_backward = nullptr;
    decltype(&sb_distill_loss) distill = nullptr;
    decltype(&sb_distill_loss_backward) distill_backward = nullptr;
    decltype(&sb_last_error) last_error = nullptr;
} api;

void bind(const std::vector<int64_t>& f) {
    TORCH_CHECK(f.size() == 5, "bind takes five addresses");
    api.logprobs = reinterpret_cast<decltype(api.logprobs)>(f[0]);
    api.logprobs_backward = reinterpret_cast<decltype(api.logprobs_backward)>(f[1]);
    api.distill = reinterpret_cast<decltype(api.distill)>(f[2]);
    api.distill_backward = reinterpret_cast<decltype(api.distill_backward)>(f[3]);
    api.last_error = reinterpret_cast<decltype(api.last_error)>(f[4]);
}

// Call f(stream) for the tensor's device and raise what it reports.
template <typename F> void launch(const Tensor& x, F f) {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const int rc = f(static_cast<void*>(c10::cuda::getCurrentCUDAStream(x.device().index()).stream()));
    TORCH_CHECK(rc == SB_OK, "libstratego_b200 error ", rc, ": ", api.last_error());
}

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SB_DTYPE_F32;
        case at::kBFloat16: return SB_DTYPE_BF16;
        case at::kHalf: return SB_DTYPE_F16;
        default: return -1;
    }
}

// Forward mode: a dual tensor need not require grad, and an output without a
// tangent would count as a constant.
bool has_tangent(const Tensor& t) {
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined();
}

void check_logits(const Tensor& x, double temperature) {
    TORCH_CHECK(dtype_code(x) >= 0, "logits must be a float32, bfloat16 or float16 tensor");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= SB_POLICY_MAX_ACTIONS,
                "logits must be [..., A] with 1 <= A <= ", SB_POLICY_MAX_ACTIONS, ", got ", x.sizes());
    TORCH_CHECK(std::isfinite(temperature) && temperature >= 1e-30 && temperature <= 1e30,
                "temperature must be between 1e-30 and 1e30, got ", temperature);
    TORCH_CHECK(!has_tangent(x), "the policy operators have no forward-mode derivatives: pass the logits' primal");
}

// [..., W] as [R, W] with the elements of a row side by side: a view where the
// strides allow one, else a copy.
Tensor as_rows(Tensor t) {
    if (t.dim() == 1) t = t.unsqueeze(0);
    else if (t.dim() != 2) t = t.reshape({-1, t.size(-1)});
    return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous();
}

struct Mask {
    Tensor t;  // undefined: none
    int kind = SB_MASK_NONE;
};

Mask mask_rows(const std::optional<Tensor>& given, const Tensor& logits) {
    if (!given.has_value() || !given->defined()) return {};
    Tensor m = *given;
    TORCH_CHECK(m.scalar_type() == at::kBool || m.scalar_type() == at::kByte, "mask must be a bool or uint8 tensor");
    TORCH_CHECK(m.device() == logits.device(), "mask is on ", m.device(), ", the logits are on ", logits.device());
    const int64_t a = logits.size(-1), bits = (a + 7) / 8;
    if (a == SB_NUM_ACTIONS && m.dim() >= 2 && m.size(-1) == SB_NUM_SQUARES && m.size(-2) == SB_NUM_SQUARES)
        m = m.flatten(-2);
    const int64_t width = m.dim() ? m.size(-1) : 0;
    const bool bytes = width == a;
    TORCH_CHECK(bytes || (width == bits && m.scalar_type() == at::kByte), "mask must be [..., ", a,
                "] bool / uint8 or [..., ", bits, "] bit-packed uint8 for ", a, " actions, got ", m.sizes(), " ",
                m.scalar_type());
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    if (m.sizes().slice(0, m.dim() - 1) != lead) {
        bool fits = m.dim() <= logits.dim();
        for (int64_t i = 1; fits && i < m.dim(); ++i) {
            const int64_t n = m.size(m.dim() - 1 - i);
            fits = n == 1 || n == logits.size(logits.dim() - 1 - i);
        }
        TORCH_CHECK(fits, "mask ", m.sizes(), " does not match logits ", logits.sizes());
        std::vector<int64_t> shape(lead.begin(), lead.end());
        shape.push_back(width);
        m = m.expand(shape);
        bool one = m.dim() > 2;  // one row for all of them stays one row
        int64_t rows = 1;
        for (int64_t i = 0; i + 1 < m.dim(); ++i) {
            rows *= m.size(i);
            one = one && (m.size(i) <= 1 || m.stride(i) == 0);
        }
        if (one) m = m.as_strided({rows, width}, {0, m.stride(-1)});
    }
    return {as_rows(m), bytes ? SB_MASK_U8 : SB_MASK_BITS};
}

Tensor index_rows(const Tensor& t, at::IntArrayRef shape, const char* what, const Tensor& logits) {
    TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt || t.scalar_type() == at::kShort, what,
                " must be an int16, int32 or int64 tensor");
    TORCH_CHECK(t.sizes() == shape, what, " must have shape ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.device() == logits.device(), what, " are on ", t.device(), ", the logits are on ", logits.device());
    return t.contiguous();
}

void check_cuda(const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "logits must be on a CUDA device (there is no CPU fallback)");
    TORCH_CHECK(api.logprobs != nullptr, "libstratego_b200 is not bound");
}

template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

sb_logits describe(const Tensor& x, const Tensor& mask, int kind, double temperature) {
    sb_logits d = {};
    d.logits = x.data_ptr();
    d.mask = ptr<const uint8_t>(mask);
    d.n_rows = x.size(0);
    d.row_stride = x.stride(0);
    d.mask_stride = mask.defined() ? mask.stride(0) : 0;
    d.n_actions = (int32_t)x.size(1);
    d.dtype = dtype_code(x);
    d.mask_kind = kind;
    d.temperature = (float)temperature;
    return d;
}

at::TensorOptions floats(const Tensor& x) { return x.options().dtype(at::kFloat).requires_grad(false); }

// A gradient per row as float32 and its stride: autograd's expanded scalars
// (of a sum or a mean) stay one element.
struct RowGrad {
    Tensor t;
    int64_t stride = 0;
    explicit RowGrad(const Tensor& g) {
        if (!g.defined()) return;
        t = g.scalar_type() == at::kFloat ? g : g.to(at::kFloat);
        if (t.stride(0) != 0 && t.stride(0) != 1) t = t.contiguous();
        stride = t.stride(0);
    }
};

// The gradient has no derivative of its own: one that is asked for raises.
Tensor first_order(Tensor grad) {
    if (!at::GradMode::is_enabled()) return grad;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the policy operators' gradients cannot be differentiated again", 1);
    return (*error)({grad.requires_grad_()})[0];
}

std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ---- log-probabilities ----------------------------------------------------------

struct LogProbs {
    Tensor entropy, logprob, top_logprob, top_action, stats;
    sb_logprobs arg = {};
};

LogProbs logprobs_forward(const Tensor& x, const sb_logits& in, const Tensor& actions, int64_t top, bool keep) {
    const int64_t r = x.size(0);
    LogProbs o;
    o.entropy = at::empty({r}, floats(x));
    if (actions.defined()) o.logprob = at::empty({r}, floats(x));
    if (top) {
        o.top_logprob = at::empty({r, top}, floats(x));
        o.top_action = at::empty({r, top}, floats(x).dtype(at::kLong));
    }
    if (keep) o.stats = at::empty({r, 2}, floats(x));
    o.arg.actions = ptr<void>(actions);
    o.arg.action_bytes = actions.defined() ? (int32_t)actions.element_size() : 0;
    o.arg.top = (int32_t)top;
    o.arg.logprob = ptr<float>(o.logprob);
    o.arg.entropy = ptr<float>(o.entropy);
    o.arg.row_stats = ptr<float>(o.stats);
    o.arg.top_action = ptr<int64_t>(o.top_action);
    o.arg.top_logprob = ptr<float>(o.top_logprob);
    if (r) launch(x, [&](void* st) { return api.logprobs(&in, &o.arg, st); });
    return o;
}

variable_list outputs_of(const LogProbs& o) {
    variable_list v = {o.entropy};
    if (o.logprob.defined()) v.push_back(o.logprob);
    if (o.top_action.defined()) {
        v.push_back(o.top_logprob);
        v.push_back(o.top_action);
    }
    return v;
}

struct LogProbsNode : torch::autograd::Function<LogProbsNode> {
    // An operand that may be missing comes as an optional: autograd takes every
    // plain tensor for one of the function's variables.
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& m, int64_t kind,
                                 const std::optional<Tensor>& act, int64_t top, double temperature) {
        const Tensor mask = m.value_or(Tensor()), actions = act.value_or(Tensor());
        const LogProbs o = logprobs_forward(x, describe(x, mask, (int)kind, temperature), actions, top, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, mask, actions, o.entropy, o.top_action, o.stats});
        ctx->saved_data["args"] = std::vector<int64_t>{kind, top};
        ctx->saved_data["temperature"] = temperature;
        if (top) ctx->mark_non_differentiable({o.top_action});
        return outputs_of(o);
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &mask = saved[1], &actions = saved[2], &entropy = saved[3], &top_action = saved[4],
                     &stats = saved[5];
        const auto args = ctx->saved_data["args"].toIntVector();
        Tensor grad = at::empty(x.sizes(), x.options().requires_grad(false));
        if (x.size(0)) {
            const bool given = actions.defined(), listed = args[1] > 0;
            const RowGrad ge(g[0]), gl(given ? g[1] : Tensor());
            Tensor gt = listed ? g[given ? 2 : 1] : Tensor();
            if (gt.defined()) gt = gt.to(at::kFloat).contiguous();
            sb_logprobs f = {};
            f.actions = ptr<void>(actions);
            f.action_bytes = given ? (int32_t)actions.element_size() : 0;
            f.top = (int32_t)args[1];
            f.entropy = ptr<float>(entropy);
            f.row_stats = ptr<float>(stats);
            f.top_action = ptr<int64_t>(top_action);
            const sb_logprobs_grad go = {ptr<float>(gl.t), ptr<float>(ge.t), ptr<float>(gt), gl.stride, ge.stride,
                                         grad.data_ptr()};
            const sb_logits in = describe(x, mask, (int)args[0], ctx->saved_data["temperature"].toDouble());
            launch(x, [&](void* st) { return api.logprobs_backward(&in, &f, &go, st); });
        }
        return {first_order(grad), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// [entropy, logprob (with actions), top_logprob and top_action (with top)]
variable_list action_logprobs(const Tensor& logits, const std::optional<Tensor>& actions,
                              const std::optional<Tensor>& mask, int64_t top, double temperature) {
    check_logits(logits, temperature);
    TORCH_CHECK(top >= 0 && top <= SB_POLICY_MAX_TOP, "top must be 0..", SB_POLICY_MAX_TOP, ", got ", top);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    const Mask m = mask_rows(mask, logits);
    Tensor act;
    if (actions.has_value() && actions->defined()) act = index_rows(*actions, lead, "actions", logits);
    check_cuda(logits);
    const Tensor x = as_rows(logits);
    variable_list out;
    if (at::GradMode::is_enabled() && x.requires_grad())
        out = LogProbsNode::apply(x, given(m.t), (int64_t)m.kind, given(act), top, temperature);
    else
        out = outputs_of(logprobs_forward(x, describe(x, m.t, m.kind, temperature), act, top, false));
    if (lead.size() != 1)
        for (Tensor& t : out) {
            std::vector<int64_t> shape(lead.begin(), lead.end());
            if (t.dim() == 2) shape.push_back(top);
            t = t.view(shape);
        }
    return out;
}

// ---- distillation -----------------------------------------------------------------

sb_distill teacher_of(const Tensor& actions, const Tensor& logits, bool tail, const Tensor& loss, const Tensor& stats) {
    sb_distill d = {};
    d.teacher_actions = actions.data_ptr();
    d.teacher_logits = logits.data_ptr();
    d.action_bytes = (int32_t)actions.element_size();
    d.teacher_dtype = dtype_code(logits);
    d.listed = (int32_t)actions.size(1);
    d.tail = tail;
    d.loss = ptr<float>(loss);
    d.row_stats = ptr<float>(stats);
    return d;
}

Tensor distill_forward(const Tensor& x, const sb_logits& in, const Tensor& ta, const Tensor& tl, bool tail, Tensor* stats) {
    Tensor loss = at::empty({x.size(0)}, floats(x));
    if (stats) *stats = at::empty({x.size(0), 6}, floats(x));
    const sb_distill d = teacher_of(ta, tl, tail, loss, stats ? *stats : Tensor());
    if (x.size(0)) launch(x, [&](void* st) { return api.distill(&in, &d, st); });
    return loss;
}

struct DistillNode : torch::autograd::Function<DistillNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& m, int64_t kind,
                          const Tensor& ta, const Tensor& tl, double temperature, bool tail) {
        const Tensor mask = m.value_or(Tensor());
        Tensor stats;
        Tensor loss = distill_forward(x, describe(x, mask, (int)kind, temperature), ta, tl, tail, &stats);
        ctx->save_for_backward({x, mask, ta, tl, stats});
        ctx->saved_data["args"] = std::vector<int64_t>{kind, tail};
        ctx->saved_data["temperature"] = temperature;
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const Tensor& x = saved[0];
        const auto args = ctx->saved_data["args"].toIntVector();
        Tensor grad = at::empty(x.sizes(), x.options().requires_grad(false));
        if (x.size(0)) {
            const RowGrad gl(g[0]);
            const sb_logits in = describe(x, saved[1], (int)args[0], ctx->saved_data["temperature"].toDouble());
            const sb_distill d = teacher_of(saved[2], saved[3], args[1] != 0, Tensor(), saved[4]);
            launch(x, [&](void* st) {
                return api.distill_backward(&in, &d, ptr<float>(gl.t), gl.stride, grad.data_ptr(), st);
            });
        }
        return {first_order(grad), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor distill_loss(const Tensor& logits, const Tensor& teacher_actions, const Tensor& teacher_logits,
                    const std::optional<Tensor>& mask, double temperature, bool tail) {
    check_logits(logits, temperature);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK(teacher_actions.dim() == logits.dim(),
                "teacher_actions must be [..., K] over the logits' leading dimensions ", lead);
    const int64_t k = teacher_actions.size(-1);
    TORCH_CHECK(k >= 1 && k <= SB_POLICY_MAX_TEACHER, "teacher_actions must list 1..", SB_POLICY_MAX_TEACHER,
                " actions per row, got ", k);
    std::vector<int64_t> shape(lead.begin(), lead.end());
    shape.push_back(k);
    Tensor ta = index_rows(teacher_actions, shape, "teacher_actions", logits);
    TORCH_CHECK(dtype_code(teacher_logits) >= 0, "teacher_logits must be a float32, bfloat16 or float16 tensor");
    TORCH_CHECK(teacher_logits.sizes() == teacher_actions.sizes() && teacher_logits.device() == logits.device(),
                "teacher_logits must be ", teacher_actions.sizes(), " on ", logits.device(), ", got ",
                teacher_logits.sizes(), " on ", teacher_logits.device());
    TORCH_CHECK(!(at::GradMode::is_enabled() && teacher_logits.requires_grad()),
                "distill_loss has no gradient for teacher_logits: detach them");
    TORCH_CHECK(!has_tangent(teacher_logits),
                "distill_loss has no forward-mode derivative for teacher_logits: pass their primal");
    const Mask m = mask_rows(mask, logits);
    check_cuda(logits);
    Tensor tl = teacher_logits.contiguous();
    if (lead.size() != 1) {
        ta = ta.view({-1, k});
        tl = tl.view({-1, k});
    }
    const Tensor x = as_rows(logits);
    Tensor loss;
    if (at::GradMode::is_enabled() && x.requires_grad())
        loss = DistillNode::apply(x, given(m.t), (int64_t)m.kind, ta, tl, temperature, tail);
    else
        loss = distill_forward(x, describe(x, m.t, m.kind, temperature), ta, tl, tail, nullptr);
    return lead.size() == 1 ? loss : loss.view(lead);
}

}  // namespace

TORCH_LIBRARY(stratego_b200, m) {
    m.def("bind(int[] entry_points) -> ()", &bind);
    m.def("action_logprobs(Tensor logits, Tensor? actions, Tensor? mask, int top, float temperature) -> Tensor[]",
          &action_logprobs);
    m.def("distill_loss(Tensor logits, Tensor teacher_actions, Tensor teacher_logits, Tensor? mask, float temperature, "
          "bool tail) -> Tensor",
          &distill_loss);
}
