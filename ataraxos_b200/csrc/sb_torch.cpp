// sb_torch.cpp -- the policy operators as torch operators with gradients.
//
// A call's arguments are checked, its outputs allocated and its kernel launched
// here, and the gradient is a node of autograd's own kind: for a small batch
// the host's work is the whole cost (a training call of 64 rows took 99 us
// through a Python autograd function, of which 50 are autograd's engine).
// The kernels stay behind the C ABI: bind() receives the addresses of its
// entry points, so this file links against torch alone.
//
// The public operators are compositions: they check and reshape, in symbolic
// sizes, and call an operator on rows (its name starts with an underscore) that
// has a CUDA and a shape-only implementation.  What traces or fakes tensors
// meets the operators on rows, one node for each launch.  A traced graph may
// hand them rows that lie otherwise than those it was traced with, so they lay
// out and check their own operands.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <type_traits>
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
    TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) >= 1 && x.sym_size(-1) <= SB_POLICY_MAX_ACTIONS,
                "logits must be [..., A] with 1 <= A <= ", SB_POLICY_MAX_ACTIONS, ", got ", x.sym_sizes());
    TORCH_CHECK(std::isfinite(temperature) && temperature >= 1e-30 && temperature <= 1e30,
                "temperature must be between 1e-30 and 1e30, got ", temperature);
    TORCH_CHECK(!has_tangent(x), "the policy operators have no forward-mode derivatives: pass the logits' primal");
}

// [R, W] with the elements of a row side by side.
Tensor side_by_side(const Tensor& t) {
    return t.sym_size(1) == 1 || t.sym_stride(1) == 1 ? t : t.contiguous();
}

// [..., W] as [R, W]: a view where the strides allow one, else a copy.
Tensor as_rows(const Tensor& t) {
    if (t.dim() == 2) return side_by_side(t);
    return side_by_side(t.dim() == 1 ? t.unsqueeze(0) : t.reshape_symint({-1, t.sym_size(-1)}));
}

struct Mask {
    std::optional<Tensor> t;
    int64_t kind = SB_MASK_NONE;
};

Mask mask_rows(const std::optional<Tensor>& given, const Tensor& logits) {
    if (!given.has_value() || !given->defined()) return {};
    Tensor m = *given;
    TORCH_CHECK(m.scalar_type() == at::kBool || m.scalar_type() == at::kByte, "mask must be a bool or uint8 tensor");
    TORCH_CHECK(m.device() == logits.device(), "mask is on ", m.device(), ", the logits are on ", logits.device());
    const c10::SymInt a = logits.sym_size(-1), bits = (a + 7) / 8;
    if (a == SB_NUM_ACTIONS && m.dim() >= 2 && m.sym_size(-1) == SB_NUM_SQUARES && m.sym_size(-2) == SB_NUM_SQUARES)
        m = m.flatten(-2);
    const c10::SymInt width = m.dim() ? m.sym_size(-1) : c10::SymInt(0);
    const bool bytes = width == a;
    TORCH_CHECK(bytes || (width == bits && m.scalar_type() == at::kByte), "mask must be [..., ", a,
                "] bool / uint8 or [..., ", bits, "] bit-packed uint8 for ", a, " actions, got ", m.sym_sizes(), " ",
                m.scalar_type());
    const auto lead = logits.sym_sizes().slice(0, logits.dim() - 1);
    if (m.sym_sizes().slice(0, m.dim() - 1) != lead) {
        bool fits = m.dim() <= logits.dim();
        for (int64_t i = 1; fits && i < m.dim(); ++i) {
            const c10::SymInt n = m.sym_size(m.dim() - 1 - i);
            fits = n == 1 || n == logits.sym_size(logits.dim() - 1 - i);
        }
        TORCH_CHECK(fits, "mask ", m.sym_sizes(), " does not match logits ", logits.sym_sizes());
        std::vector<c10::SymInt> shape(lead.begin(), lead.end());
        shape.push_back(width);
        m = m.expand_symint(shape);
        bool one = m.dim() > 2;  // one row for all of them stays one row
        c10::SymInt rows = 1;
        for (int64_t i = 0; i + 1 < m.dim(); ++i) {
            rows *= m.sym_size(i);
            one = one && (m.sym_size(i) <= 1 || m.sym_stride(i) == 0);
        }
        if (one) m = m.as_strided_symint({rows, width}, {0, m.sym_stride(-1)});
    }
    return {as_rows(m), bytes ? SB_MASK_U8 : SB_MASK_BITS};
}

void check_index(const Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt || t.scalar_type() == at::kShort, what,
                " must be an int16, int32 or int64 tensor");
}

Tensor index_rows(const Tensor& t, c10::SymIntArrayRef shape, const char* what, const Tensor& logits) {
    check_index(t, what);
    TORCH_CHECK(t.sym_sizes() == shape, what, " must have shape ", shape, ", got ", t.sym_sizes());
    TORCH_CHECK(t.device() == logits.device(), what, " are on ", t.device(), ", the logits are on ", logits.device());
    return t.contiguous();
}

void check_cuda(const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "logits must be on a CUDA device (there is no CPU fallback)");
    TORCH_CHECK(api.logprobs != nullptr, "libstratego_b200 is not bound");
}

template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

at::TensorOptions floats(const Tensor& x) { return x.options().dtype(at::kFloat).requires_grad(false); }

std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// The gradient has no derivative of its own: one that is asked for raises.
Tensor first_order(Tensor grad) {
    if (!at::GradMode::is_enabled()) return grad;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the policy operators' gradients cannot be differentiated again", 1);
    return (*error)({grad.requires_grad_()})[0];
}

// ---- operands of the operators on rows -------------------------------------------

// The logits and masks of a launch, each row's elements side by side.
struct Rows {
    Tensor x, mask;
    sb_logits arg = {};
    Rows(const Tensor& logits, const std::optional<Tensor>& m, int64_t kind, double temperature) {
        check_cuda(logits);
        TORCH_CHECK(logits.dim() == 2 && dtype_code(logits) >= 0, "logits must be rows of a float type");
        x = side_by_side(logits);
        if (m.has_value()) {
            TORCH_CHECK(m->dim() == 2 && m->size(0) == x.size(0) && m->element_size() == 1 && m->device() == x.device() &&
                            (kind == SB_MASK_U8 ? m->size(1) == x.size(1)
                                                : kind == SB_MASK_BITS && m->size(1) == (x.size(1) + 7) / 8),
                        "mask rows ", m->sizes(), " do not match logits ", x.sizes());
            mask = side_by_side(*m);
        }
        arg.logits = x.data_ptr();
        arg.mask = ptr<const uint8_t>(mask);
        arg.n_rows = x.size(0);
        arg.row_stride = x.stride(0);
        arg.mask_stride = mask.defined() ? mask.stride(0) : 0;
        arg.n_actions = (int32_t)x.size(1);
        arg.dtype = dtype_code(x);
        arg.mask_kind = (int32_t)kind;
        arg.temperature = (float)temperature;
    }
    // `t`, `width` elements for each row, as the kernels read it.
    Tensor beside(const Tensor& t, int64_t width, const char* what) const {
        TORCH_CHECK(t.device() == x.device() && t.numel() == x.size(0) * width, what, " do not match logits ", x.sizes());
        return t.contiguous();
    }
    Tensor beside(const Tensor& t, int64_t width, at::ScalarType type, const char* what) const {
        TORCH_CHECK(t.scalar_type() == type, what, " must be ", type, ", got ", t.scalar_type());
        return beside(t, width, what);
    }
    Tensor indices(const Tensor& t, int64_t width, const char* what) const {
        check_index(t, what);
        return beside(t, width, what);
    }
};

// A gradient per row as float32 and its stride: autograd's expanded scalars
// (of a sum or a mean) stay one element.
struct RowGrad {
    Tensor t;
    int64_t stride = 0;
    RowGrad(const Rows& rows, const Tensor& g) {
        if (!g.defined()) return;
        TORCH_CHECK(g.dim() == 1 && g.size(0) == rows.x.size(0) && g.device() == rows.x.device(),
                    "gradients do not match logits ", rows.x.sizes());
        t = g.scalar_type() == at::kFloat ? g : g.to(at::kFloat);
        if (t.stride(0) != 0 && t.stride(0) != 1) t = t.contiguous();
        stride = t.stride(0);
    }
};

// A function's registered operator, called past autograd (what calls it is the gradient's node, or needs none).
template <auto* F> const auto& op(const char* name) {
    static const auto handle =
        c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<std::remove_pointer_t<decltype(F)>>();
    return handle;
}

// ---- log-probabilities ----------------------------------------------------------

// [entropy, logprob (with actions), top_logprob and top_action (with top), row statistics (with keep)]
variable_list logprobs_outputs(const Tensor& x, bool actions, int64_t top, bool keep) {
    const c10::SymInt r = x.sym_size(0);
    variable_list o;
    o.reserve(5);
    o.push_back(at::empty_symint({r}, floats(x)));
    if (actions) o.push_back(at::empty_symint({r}, floats(x)));
    if (top) {
        o.push_back(at::empty_symint({r, top}, floats(x)));
        o.push_back(at::empty_symint({r, top}, floats(x).dtype(at::kLong)));
    }
    if (keep) o.push_back(at::empty_symint({r, 2}, floats(x)));
    return o;
}

variable_list logprobs_rows_meta(const Tensor& x, const std::optional<Tensor>& actions, const std::optional<Tensor>&,
                                 int64_t, int64_t top, double, bool keep) {
    return logprobs_outputs(x, actions.has_value(), top, keep);
}

variable_list logprobs_rows(const Tensor& logits, const std::optional<Tensor>& actions, const std::optional<Tensor>& mask,
                            int64_t kind, int64_t top, double temperature, bool keep) {
    const Rows rows(logits, mask, kind, temperature);
    Tensor act;
    sb_logprobs arg = {};
    if (actions.has_value()) {
        act = rows.indices(*actions, 1, "actions");
        arg.actions = act.data_ptr();
        arg.action_bytes = (int32_t)act.element_size();
    }
    variable_list out = logprobs_outputs(rows.x, act.defined(), top, keep);
    size_t i = 0;
    arg.top = (int32_t)top;
    arg.entropy = ptr<float>(out[i++]);
    if (act.defined()) arg.logprob = ptr<float>(out[i++]);
    if (top) {
        arg.top_logprob = ptr<float>(out[i++]);
        arg.top_action = ptr<int64_t>(out[i++]);
    }
    if (keep) arg.row_stats = ptr<float>(out[i]);
    if (rows.arg.n_rows) launch(rows.x, [&](void* st) { return api.logprobs(&rows.arg, &arg, st); });
    return out;
}

Tensor logprobs_rows_backward_meta(const Tensor& x, const std::optional<Tensor>&, const std::optional<Tensor>&, int64_t,
                                   const std::optional<Tensor>&, const Tensor&, const Tensor&,
                                   const std::optional<Tensor>&, const std::optional<Tensor>&,
                                   const std::optional<Tensor>&, double) {
    return at::empty_symint(x.sym_sizes(), x.options().requires_grad(false));
}

Tensor logprobs_rows_backward(const Tensor& logits, const std::optional<Tensor>& actions, const std::optional<Tensor>& mask,
                              int64_t kind, const std::optional<Tensor>& top_action, const Tensor& entropy,
                              const Tensor& row_stats, const std::optional<Tensor>& g_entropy,
                              const std::optional<Tensor>& g_logprob, const std::optional<Tensor>& g_top,
                              double temperature) {
    const Rows rows(logits, mask, kind, temperature);
    Tensor grad = at::empty(rows.x.sizes(), rows.x.options().requires_grad(false));
    Tensor act, top, gt;
    sb_logprobs f = {};
    if (actions.has_value()) {
        act = rows.indices(*actions, 1, "actions");
        f.actions = act.data_ptr();
        f.action_bytes = (int32_t)act.element_size();
    }
    if (top_action.has_value()) {
        f.top = (int32_t)top_action->size(-1);
        top = rows.beside(*top_action, f.top, at::kLong, "alternatives");
        f.top_action = ptr<int64_t>(top);
        if (g_top.has_value()) gt = rows.beside(*g_top, f.top, "gradients").to(at::kFloat);
    }
    const Tensor h = rows.beside(entropy, 1, at::kFloat, "entropies"),
                 stats = rows.beside(row_stats, 2, at::kFloat, "statistics");
    f.entropy = ptr<float>(h);
    f.row_stats = ptr<float>(stats);
    const RowGrad ge(rows, g_entropy.value_or(Tensor())), gl(rows, g_logprob.value_or(Tensor()));
    const sb_logprobs_grad g = {ptr<float>(gl.t), ptr<float>(ge.t), ptr<float>(gt), gl.stride, ge.stride, grad.data_ptr()};
    if (rows.arg.n_rows) launch(rows.x, [&](void* st) { return api.logprobs_backward(&rows.arg, &f, &g, st); });
    return grad;
}

variable_list call_logprobs(const Tensor& x, const std::optional<Tensor>& actions, const std::optional<Tensor>& mask,
                            int64_t kind, int64_t top, double temperature, bool keep) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    return op<&logprobs_rows>("stratego_b200::_action_logprobs").call(x, actions, mask, kind, top, temperature, keep);
}

struct LogProbsNode : torch::autograd::Function<LogProbsNode> {
    // An operand that may be missing comes as an optional: autograd takes every
    // plain tensor for one of the function's variables.
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& m, int64_t kind,
                                 const std::optional<Tensor>& act, int64_t top, double temperature) {
        variable_list out = call_logprobs(x, act, m, kind, top, temperature, true);
        const Tensor stats = out.back();
        out.pop_back();
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, m.value_or(Tensor()), act.value_or(Tensor()), out[0], top ? out.back() : Tensor(), stats});
        ctx->saved_data["kind"] = kind;
        ctx->saved_data["temperature"] = temperature;
        if (top) ctx->mark_non_differentiable({out.back()});
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const bool actions = saved[2].defined(), top = saved[4].defined();
        Tensor grad;
        {
            const at::AutoDispatchBelowADInplaceOrView guard;
            grad = op<&logprobs_rows_backward>("stratego_b200::_action_logprobs_backward")
                       .call(saved[0], given(saved[2]), given(saved[1]), ctx->saved_data["kind"].toInt(), given(saved[4]),
                             saved[3], saved[5], given(g[0]), given(actions ? g[1] : Tensor()),
                             given(top ? g[actions ? 2 : 1] : Tensor()), ctx->saved_data["temperature"].toDouble());
        }
        return {first_order(grad), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// [entropy, logprob (with actions), top_logprob and top_action (with top)]
variable_list action_logprobs(const Tensor& logits, const std::optional<Tensor>& actions,
                              const std::optional<Tensor>& mask, int64_t top, double temperature) {
    check_logits(logits, temperature);
    TORCH_CHECK(top >= 0 && top <= SB_POLICY_MAX_TOP, "top must be 0..", SB_POLICY_MAX_TOP, ", got ", top);
    const auto lead = logits.sym_sizes().slice(0, logits.dim() - 1);
    const Mask m = mask_rows(mask, logits);
    std::optional<Tensor> act;
    if (actions.has_value() && actions->defined()) act = index_rows(*actions, lead, "actions", logits);
    check_cuda(logits);
    const Tensor x = as_rows(logits);
    variable_list out;
    if (at::GradMode::is_enabled() && x.requires_grad())
        out = LogProbsNode::apply(x, m.t, m.kind, act, top, temperature);
    else
        out = call_logprobs(x, act, m.t, m.kind, top, temperature, false);
    if (lead.size() != 1)
        for (Tensor& t : out) {
            std::vector<c10::SymInt> shape(lead.begin(), lead.end());
            if (t.dim() == 2) shape.push_back(top);
            t = t.view_symint(shape);
        }
    return out;
}

// ---- distillation -----------------------------------------------------------------

// A launch's teacher; `ta` and `tl` keep its operands alive.
struct Teacher {
    Tensor ta, tl;
    sb_distill arg = {};
    Teacher(const Rows& rows, const Tensor& actions, const Tensor& logits, bool tail) {
        TORCH_CHECK(actions.dim() == 2 && dtype_code(logits) >= 0, "the teacher must be rows of actions and floats");
        ta = rows.indices(actions, actions.size(1), "teacher_actions");
        tl = rows.beside(logits, actions.size(1), "teacher_logits");
        arg.teacher_actions = ta.data_ptr();
        arg.teacher_logits = tl.data_ptr();
        arg.action_bytes = (int32_t)ta.element_size();
        arg.teacher_dtype = dtype_code(tl);
        arg.listed = (int32_t)ta.size(1);
        arg.tail = tail;
    }
};

// [loss, row statistics (with keep)]
variable_list distill_outputs(const Tensor& x, bool keep) {
    variable_list o;
    o.reserve(2);
    o.push_back(at::empty_symint({x.sym_size(0)}, floats(x)));
    if (keep) o.push_back(at::empty_symint({x.sym_size(0), 6}, floats(x)));
    return o;
}

variable_list distill_rows_meta(const Tensor& x, const Tensor&, const Tensor&, const std::optional<Tensor>&, int64_t, double,
                                bool, bool keep) {
    return distill_outputs(x, keep);
}

variable_list distill_rows(const Tensor& logits, const Tensor& teacher_actions, const Tensor& teacher_logits,
                           const std::optional<Tensor>& mask, int64_t kind, double temperature, bool tail, bool keep) {
    const Rows rows(logits, mask, kind, temperature);
    Teacher t(rows, teacher_actions, teacher_logits, tail);
    variable_list out = distill_outputs(rows.x, keep);
    t.arg.loss = ptr<float>(out[0]);
    if (keep) t.arg.row_stats = ptr<float>(out[1]);
    if (rows.arg.n_rows) launch(rows.x, [&](void* st) { return api.distill(&rows.arg, &t.arg, st); });
    return out;
}

Tensor distill_rows_backward_meta(const Tensor& x, const Tensor&, const Tensor&, const std::optional<Tensor>&, int64_t,
                                  const Tensor&, const Tensor&, double, bool) {
    return at::empty_symint(x.sym_sizes(), x.options().requires_grad(false));
}

Tensor distill_rows_backward(const Tensor& logits, const Tensor& teacher_actions, const Tensor& teacher_logits,
                             const std::optional<Tensor>& mask, int64_t kind, const Tensor& row_stats,
                             const Tensor& g_loss, double temperature, bool tail) {
    const Rows rows(logits, mask, kind, temperature);
    Teacher t(rows, teacher_actions, teacher_logits, tail);
    Tensor grad = at::empty(rows.x.sizes(), rows.x.options().requires_grad(false));
    const Tensor stats = rows.beside(row_stats, 6, at::kFloat, "statistics");
    t.arg.row_stats = ptr<float>(stats);
    const RowGrad g(rows, g_loss);
    if (rows.arg.n_rows)
        launch(rows.x, [&](void* st) {
            return api.distill_backward(&rows.arg, &t.arg, ptr<float>(g.t), g.stride, grad.data_ptr(), st);
        });
    return grad;
}

variable_list call_distill(const Tensor& x, const Tensor& ta, const Tensor& tl, const std::optional<Tensor>& mask,
                           int64_t kind, double temperature, bool tail, bool keep) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    return op<&distill_rows>("stratego_b200::_distill_loss").call(x, ta, tl, mask, kind, temperature, tail, keep);
}

struct DistillNode : torch::autograd::Function<DistillNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& m, int64_t kind,
                          const Tensor& ta, const Tensor& tl, double temperature, bool tail) {
        const variable_list out = call_distill(x, ta, tl, m, kind, temperature, tail, true);
        ctx->save_for_backward({x, m.value_or(Tensor()), ta, tl, out[1]});
        ctx->saved_data["kind"] = kind;
        ctx->saved_data["tail"] = tail;
        ctx->saved_data["temperature"] = temperature;
        return out[0];
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        Tensor grad;
        {
            const at::AutoDispatchBelowADInplaceOrView guard;
            grad = op<&distill_rows_backward>("stratego_b200::_distill_loss_backward")
                       .call(saved[0], saved[2], saved[3], given(saved[1]), ctx->saved_data["kind"].toInt(), saved[4], g[0],
                             ctx->saved_data["temperature"].toDouble(), ctx->saved_data["tail"].toBool());
        }
        return {first_order(grad), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor distill_loss(const Tensor& logits, const Tensor& teacher_actions, const Tensor& teacher_logits,
                    const std::optional<Tensor>& mask, double temperature, bool tail) {
    check_logits(logits, temperature);
    const auto lead = logits.sym_sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK(teacher_actions.dim() == logits.dim(),
                "teacher_actions must be [..., K] over the logits' leading dimensions ", lead);
    const c10::SymInt k = teacher_actions.sym_size(-1);
    TORCH_CHECK(k >= 1 && k <= SB_POLICY_MAX_TEACHER, "teacher_actions must list 1..", SB_POLICY_MAX_TEACHER,
                " actions per row, got ", k);
    std::vector<c10::SymInt> shape(lead.begin(), lead.end());
    shape.push_back(k);
    Tensor ta = index_rows(teacher_actions, shape, "teacher_actions", logits);
    TORCH_CHECK(dtype_code(teacher_logits) >= 0, "teacher_logits must be a float32, bfloat16 or float16 tensor");
    TORCH_CHECK(teacher_logits.sym_sizes() == teacher_actions.sym_sizes() && teacher_logits.device() == logits.device(),
                "teacher_logits must be ", teacher_actions.sym_sizes(), " on ", logits.device(), ", got ",
                teacher_logits.sym_sizes(), " on ", teacher_logits.device());
    TORCH_CHECK(!(at::GradMode::is_enabled() && teacher_logits.requires_grad()),
                "distill_loss has no gradient for teacher_logits: detach them");
    TORCH_CHECK(!has_tangent(teacher_logits),
                "distill_loss has no forward-mode derivative for teacher_logits: pass their primal");
    const Mask m = mask_rows(mask, logits);
    check_cuda(logits);
    Tensor tl = teacher_logits.contiguous();
    if (lead.size() != 1) {
        ta = ta.view_symint({-1, k});
        tl = tl.view_symint({-1, k});
    }
    const Tensor x = as_rows(logits);
    Tensor loss;
    if (at::GradMode::is_enabled() && x.requires_grad())
        loss = DistillNode::apply(x, m.t, m.kind, ta, tl, temperature, tail);
    else
        loss = call_distill(x, ta, tl, m.t, m.kind, temperature, tail, false)[0];
    return lead.size() == 1 ? loss : loss.view_symint(lead);
}

}  // namespace

TORCH_LIBRARY(stratego_b200, m) {
    m.def("bind(int[] entry_points) -> ()", &bind);
    m.def("action_logprobs(Tensor logits, Tensor? actions, Tensor? mask, int top, float temperature) -> Tensor[]",
          &action_logprobs);
    m.def("distill_loss(Tensor logits, Tensor teacher_actions, Tensor teacher_logits, Tensor? mask, float temperature, "
          "bool tail) -> Tensor",
          &distill_loss);
    m.def("_action_logprobs(Tensor logits, Tensor? actions, Tensor? mask, int mask_kind, int top, float temperature, "
          "bool keep) -> Tensor[]");
    m.def("_action_logprobs_backward(Tensor logits, Tensor? actions, Tensor? mask, int mask_kind, Tensor? top_action, "
          "Tensor entropy, Tensor row_stats, Tensor? g_entropy, Tensor? g_logprob, Tensor? g_top, float temperature) "
          "-> Tensor");
    m.def("_distill_loss(Tensor logits, Tensor teacher_actions, Tensor teacher_logits, Tensor? mask, int mask_kind, "
          "float temperature, bool tail, bool keep) -> Tensor[]");
    m.def("_distill_loss_backward(Tensor logits, Tensor teacher_actions, Tensor teacher_logits, Tensor? mask, "
          "int mask_kind, Tensor row_stats, Tensor g_loss, float temperature, bool tail) -> Tensor");
}

TORCH_LIBRARY_IMPL(stratego_b200, CUDA, m) {
    m.impl("_action_logprobs", &logprobs_rows);
    m.impl("_action_logprobs_backward", &logprobs_rows_backward);
    m.impl("_distill_loss", &distill_rows);
    m.impl("_distill_loss_backward", &distill_rows_backward);
}

// A graph that was traced without gradients calls these with logits that require some: its backward pass raises.
TORCH_LIBRARY_IMPL(stratego_b200, Autograd, m) {
    for (const char* name : {"_action_logprobs", "_action_logprobs_backward", "_distill_loss", "_distill_loss_backward"})
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(stratego_b200, Meta, m) {
    m.impl("_action_logprobs", &logprobs_rows_meta);
    m.impl("_action_logprobs_backward", &logprobs_rows_backward_meta);
    m.impl("_distill_loss", &distill_rows_meta);
    m.impl("_distill_loss_backward", &distill_rows_backward_meta);
}
