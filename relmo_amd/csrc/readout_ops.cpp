// Torch binding of the readout ops (the relm_mp namespace's second part; the
// message-passing ops are in relm_mp_ops.cpp).  No reference counterpart: what a
// program runs on the object states that the message passing leaves.  GPU tensors
// of float32, bfloat16 or float16 (the facade runs ATen formulations for CPU
// tensors).  The ops that have gradients make their autograd nodes here: a call's
// host time counts beside kernels of a few microseconds.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <limits>
#include <memory>
#include <mutex>
#include <optional>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "relm_mp.h"

namespace relm_amd {
namespace readout {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The ops have no forward-mode formula.  A tangent does not need requires_grad (nor grad mode),
// so every call looks for one: the result would leave it out.
void refuse_tangents(std::initializer_list<const Tensor*> tensors, const char* op) {
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op, ": no forward-mode derivative is implemented.");
}

// Gradients that are themselves not differentiated: with create_graph, differentiating
// them raises.
variable_list once(variable_list grads, const char* op) {
    if (!at::GradMode::is_enabled()) return grads;
    auto stop = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate twice the backward of ") + op + ", which has no second derivative",
        static_cast<int64_t>(grads.size()));
    variable_list in;
    for (Tensor& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
    return (*stop)(std::move(in));
}

void raise_if(int rc) { TORCH_CHECK(rc == RELM_MP_OK, relm_mp_last_error()); }

hipStream_t current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int value_dtype(const Tensor& t, const char* op, const char* name) {
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a GPU tensor.");
    switch (t.scalar_type()) {
        case at::kFloat: return RELM_MP_F32;
        case at::kBFloat16: return RELM_MP_BF16;
        case at::kHalf: return RELM_MP_F16;
        default: TORCH_CHECK(false, op, ": ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type(), ".");
    }
}

void check_like(const Tensor& t, const Tensor& like, const char* op, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type() && t.device() == like.device(), op, ": ", name,
                " must have the dtype and the device of the first argument.");
}

void check_same(const Tensor& t, const Tensor& like, const char* op, const char* name) {
    check_like(t, like, op, name);
    TORCH_CHECK_VALUE(t.sizes() == like.sizes(), op, ": ", name, " must have the shape of the first argument.");
}

Tensor bytes(size_t n, const Tensor& like) {
    return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

const void* opt_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// ---- residual norm -------------------------------------------------------------

struct NormArgs {
    int dtype;
    Tensor x, r, w;
    int64_t rows, width;
};

NormArgs norm_args(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, const char* op) {
    NormArgs a{value_dtype(x, op, "x"), x.contiguous(), Tensor(), weight.contiguous(), 0, 0};
    TORCH_CHECK_VALUE(x.dim() >= 1, op, ": x must have at least one dimension.");
    a.width = x.size(-1);
    a.rows = a.width == 0 ? 0 : x.numel() / a.width;
    check_like(weight, x, op, "weight");
    TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == a.width, op, ": weight must be [", a.width, "].");
    if (residual.has_value() && residual->defined()) {
        check_same(*residual, x, op, "residual");
        a.r = residual->contiguous();
    }
    return a;
}

struct NormResult {
    Tensor y, h, rstd;  // h: only with a residual (else it is x); rstd: only if kept
};

NormResult norm_forward(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps, bool keep) {
    const NormArgs a = norm_args(x, residual, weight, "add_rms_norm");
    c10::OptionalDeviceGuard guard(x.device());
    NormResult o;
    o.y = at::empty(x.sizes(), a.x.options());
    if (a.r.defined()) o.h = at::empty(x.sizes(), a.x.options());
    if (keep) o.rstd = at::empty({a.rows}, a.x.options().dtype(at::kFloat));
    raise_if(relm_mp_add_rms_norm(a.dtype, a.x.const_data_ptr(), opt_ptr(a.r), a.w.const_data_ptr(), a.rows, a.width,
                                  static_cast<float>(eps), o.y.data_ptr(), a.r.defined() ? o.h.data_ptr() : nullptr,
                                  keep ? o.rstd.data_ptr<float>() : nullptr, current_stream(x)));
    return o;
}

// (dx, dweight) from the gradients of y and, where defined, of h.
std::tuple<Tensor, Tensor> norm_backward(const Tensor& grad_y, const Tensor& grad_h, const Tensor& h, const Tensor& weight,
                                         const Tensor& rstd) {
    const NormArgs a = norm_args(h, std::nullopt, weight, "add_rms_norm backward");
    const Tensor gy = grad_y.contiguous(), gh = grad_h.defined() ? grad_h.contiguous() : Tensor();
    c10::OptionalDeviceGuard guard(h.device());
    Tensor dx = at::empty(h.sizes(), a.x.options());
    Tensor dw = at::empty(weight.sizes(), a.x.options());
    const size_t need = relm_mp_add_rms_norm_backward_workspace_size(a.dtype, a.rows, a.width);
    const Tensor ws = bytes(need, h);
    raise_if(relm_mp_add_rms_norm_backward(a.dtype, gy.const_data_ptr(), opt_ptr(gh), a.x.const_data_ptr(),
                                           a.w.const_data_ptr(), rstd.const_data_ptr<float>(), a.rows, a.width, dx.data_ptr(),
                                           dw.data_ptr(), ws.data_ptr(), need, current_stream(h)));
    return {dx, dw};
}

// (y, h); the backward reads h, rounded as it was stored, and the rows' 1 / root.
struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& weight,
                                 double eps) {
        const NormResult o = norm_forward(x, residual, weight, eps, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({o.h, weight, o.rstd});
        return {o.y, o.h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        if (!grads[0].defined()) return {grads[1], grads[1], Tensor(), Tensor()};
        refuse_tangents({&grads[0], &grads[1]}, "add_rms_norm backward");
        const auto [dx, dw] = norm_backward(grads[0], grads[1], saved[0], saved[1], saved[2]);
        return once({dx, dx, dw, Tensor()}, "add_rms_norm");
    }
};

struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, double eps) {
        const NormResult o = norm_forward(x, std::nullopt, weight, eps, true);
        ctx->save_for_backward({x, weight, o.rstd});
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        refuse_tangents({&grads[0]}, "rms_norm backward");
        const auto [dx, dw] = norm_backward(grads[0], Tensor(), saved[0], saved[1], saved[2]);
        return once({dx, dw, Tensor()}, "rms_norm");
    }
};

}  // namespace

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
    refuse_tangents({&x, &residual, &weight}, "add_rms_norm");
    if (wants_grad({&x, &residual, &weight})) {
        const variable_list o = AddRmsNorm::apply(x, residual, weight, eps);
        return {o[0], o[1]};
    }
    const NormResult o = norm_forward(x, residual, weight, eps, false);
    return {o.y, o.h};
}

Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps) {
    refuse_tangents({&x, &weight}, "rms_norm");
    if (wants_grad({&x, &weight})) return RmsNorm::apply(x, weight, eps);
    return norm_forward(x, std::nullopt, weight, eps, false).y;
}

// (q, scale, h); without a residual h is empty (it would be x).
std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8(const Tensor& x, const std::optional<Tensor>& residual,
                                                    const Tensor& weight, double eps) {
    refuse_tangents({&x, &weight}, "add_rms_norm_fp8");
    if (residual.has_value()) refuse_tangents({&*residual}, "add_rms_norm_fp8");
    const NormArgs a = norm_args(x, residual, weight, "add_rms_norm_fp8");
    c10::OptionalDeviceGuard guard(x.device());
    Tensor q = at::empty(x.sizes(), a.x.options().dtype(at::kFloat8_e4m3fn));
    Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), a.x.options().dtype(at::kFloat));
    if (a.width == 0) scale.fill_(1.0);
    Tensor h = a.r.defined() ? at::empty(x.sizes(), a.x.options()) : at::empty({0}, a.x.options());
    raise_if(relm_mp_add_rms_norm_fp8(a.dtype, a.x.const_data_ptr(), opt_ptr(a.r), a.w.const_data_ptr(), a.rows, a.width,
                                      static_cast<float>(eps), q.data_ptr(), scale.data_ptr<float>(),
                                      a.r.defined() ? h.data_ptr() : nullptr, current_stream(x)));
    return {q, scale, h};
}

// ---- cross attention -------------------------------------------------------------

// A batch's plan with its table on the device.  The table is copied there before the
// constructor returns, so any stream may use it; a stream other than the one the
// memory was allocated on is recorded with the allocator.
//
// Ops take a plan by its number: an argument of a class would send every call through
// Python's dispatch of such arguments (8 us).  The list holds no plan alive; a number
// whose plan is gone, or that never was, is refused.
void forget_plan(int64_t number);

struct AttentionPlan : torch::CustomClassHolder {
    relm_mp_attention_plan plan{};
    Tensor table;
    hipStream_t stream = nullptr;
    int64_t number = 0;

    void release_resources() override { forget_plan(number); }

    void used_on(const c10::hip::HIPStream& s) const {
        if (table.numel() > 0 && s.stream() != stream)
            c10::hip::HIPCachingAllocator::recordStream(table.storage().data_ptr(), s);
    }
};

struct PlanList {
    std::mutex lock;
    std::unordered_map<int64_t, c10::weak_intrusive_ptr<AttentionPlan>> plans;
    int64_t next = 1;
};
PlanList& plan_list() {
    static PlanList* list = new PlanList;  // outlives plans that Python frees at exit
    return *list;
}

void forget_plan(int64_t number) {
    PlanList& list = plan_list();
    const std::lock_guard<std::mutex> hold(list.lock);
    list.plans.erase(number);
}

c10::intrusive_ptr<AttentionPlan> plan_of(int64_t number, const char* op) {
    PlanList& list = plan_list();
    const std::lock_guard<std::mutex> hold(list.lock);
    const auto at = list.plans.find(number);
    auto plan = at == list.plans.end() ? c10::intrusive_ptr<AttentionPlan>() : at->second.lock();
    TORCH_CHECK_VALUE(plan, op, ": the plan no longer exists.");
    return plan;
}

// The plan, its number, and the offsets it was made from ([2, graphs + 1], in host memory).
std::tuple<c10::intrusive_ptr<AttentionPlan>, int64_t, Tensor> attention_plan(const Tensor& q_offsets, const Tensor& k_offsets,
                                                                              int64_t heads, int64_t kv_heads) {
    for (const Tensor* t : {&q_offsets, &k_offsets})
        TORCH_CHECK(t->dim() == 1 && t->scalar_type() == at::kLong && t->is_cuda() && t->numel() >= 1 &&
                        t->device() == q_offsets.device() && t->numel() == q_offsets.numel(),
                    "attention_plan: q_offsets and k_offsets must be int64 [graphs + 1] on one GPU.");
    TORCH_CHECK(heads >= 1 && heads <= 4096 && kv_heads >= 1 && kv_heads <= 4096,
                "attention_plan: heads and kv_heads must be in [1, 4096].");
    c10::OptionalDeviceGuard guard(q_offsets.device());
    const Tensor host = at::stack({q_offsets, k_offsets}).cpu();  // one copy, waited for
    const int64_t graphs = q_offsets.numel() - 1;
    const int64_t* qo = host.const_data_ptr<int64_t>();
    const int64_t* ko = qo + graphs + 1;
    auto ref = c10::make_intrusive<AttentionPlan>();
    const auto build = [&](const Tensor& table) {
        return relm_mp_attention_plan_build(qo, ko, graphs, qo[graphs], ko[graphs], static_cast<int32_t>(heads),
                                            static_cast<int32_t>(kv_heads), table.data_ptr(),
                                            static_cast<size_t>(table.numel()), &ref->plan);
    };
    Tensor table = at::empty({4096 + 512 * graphs}, at::kByte);  // enough for 16 records to a graph
    int rc = build(table);
    if (rc == RELM_MP_ERR_WORKSPACE) {
        table = at::empty({ref->plan.table_bytes}, at::kByte);
        rc = build(table);
    }
    raise_if(rc);
    table = table.narrow(0, 0, ref->plan.table_bytes);
    const auto s = c10::hip::getCurrentHIPStream(q_offsets.get_device());
    ref->table = table.to(q_offsets.device());
    ref->stream = s.stream();
    ref->plan.table = ref->plan.table_bytes > 0 ? ref->table.const_data_ptr() : nullptr;
    PlanList& list = plan_list();
    const std::lock_guard<std::mutex> hold(list.lock);
    ref->number = list.next++;
    list.plans.emplace(ref->number, c10::weak_intrusive_ptr<AttentionPlan>(ref));
    return {ref, ref->number, host};
}

namespace {

// [rows, heads, dim] with unit strides of the values, or a copy that has them.
Tensor with_unit_values(const Tensor& t) { return t.stride(2) == 1 || t.size(2) <= 1 ? t : t.contiguous(); }

relm_mp_head_rows head_rows(const Tensor& t) { return {t.const_data_ptr(), t.stride(0), t.stride(1)}; }

struct AttnArgs {
    int dtype;
    Tensor q, k, v, mask;
    int64_t dim;
    float scale;
    const uint8_t* mask_ptr() const {
        return mask.defined() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr;
    }
};

AttnArgs attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionPlan& p, const Tensor& key_mask,
                        double scale) {
    const char* op = "cross_attention";
    AttnArgs a;
    a.dtype = value_dtype(q, op, "q");
    for (const Tensor* t : {&q, &k, &v}) {
        TORCH_CHECK_VALUE(t->dim() == 3, op, ": q, k and v must be [rows, heads, head_dim].");
        check_like(*t, q, op, "k and v");
    }
    a.dim = q.size(2);
    TORCH_CHECK_VALUE(a.dim >= 1 && a.dim <= RELM_MP_MAX_HEAD_DIM, op, ": head_dim must be in [1, ", RELM_MP_MAX_HEAD_DIM,
                      "].");
    TORCH_CHECK_VALUE(q.size(0) == p.plan.q_rows && q.size(1) == p.plan.heads, op, ": q must be [", p.plan.q_rows, ", ",
                      p.plan.heads, ", head_dim] for this plan.");
    for (const Tensor* t : {&k, &v})
        TORCH_CHECK_VALUE(t->size(0) == p.plan.k_rows && t->size(1) == p.plan.kv_heads && t->size(2) == a.dim, op,
                          ": k and v must be [", p.plan.k_rows, ", ", p.plan.kv_heads, ", ", a.dim, "] for this plan.");
    TORCH_CHECK_VALUE(p.table.device() == q.device(), op, ": the plan is on another device.");
    a.q = with_unit_values(q);
    a.k = with_unit_values(k);
    a.v = with_unit_values(v);
    if (key_mask.defined()) {
        TORCH_CHECK_VALUE(key_mask.dim() == 1 && key_mask.size(0) == p.plan.k_rows && key_mask.scalar_type() == at::kBool &&
                              key_mask.device() == q.device(),
                          op, ": key_mask must be bool [", p.plan.k_rows, "] on the device of q.");
        a.mask = key_mask.contiguous();
    }
    a.scale = static_cast<float>(scale);
    TORCH_CHECK_VALUE(a.scale > 0.0f && a.scale < std::numeric_limits<float>::infinity(), op,
                      ": scale must be finite and positive.");
    return a;
}

// (out, stats); stats only if kept.
std::tuple<Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionPlan& plan,
                                             const Tensor& key_mask, double scale, bool keep) {
    const AttnArgs a = attention_args(q, k, v, plan, key_mask, scale);
    c10::OptionalDeviceGuard guard(q.device());
    const auto stream = c10::hip::getCurrentHIPStream(q.get_device());
    plan.used_on(stream);
    Tensor out = at::empty(q.sizes(), q.options()), stats;
    if (keep) stats = at::empty({q.size(0), q.size(1), 2}, q.options().dtype(at::kFloat));
    const size_t need = relm_mp_cross_attention_workspace_size(&plan.plan, a.dim);
    const Tensor ws = need > 0 ? bytes(need, q) : Tensor();
    const relm_mp_head_rows qr = head_rows(a.q), kr = head_rows(a.k), vr = head_rows(a.v);
    void* const wp = need > 0 ? ws.data_ptr() : nullptr;
    if (keep)
        raise_if(relm_mp_cross_attention_keep(a.dtype, &plan.plan, &qr, &kr, &vr, a.dim, a.mask_ptr(), a.scale, out.data_ptr(),
                                              stats.data_ptr<float>(), wp, need, stream.stream()));
    else
        raise_if(relm_mp_cross_attention(a.dtype, &plan.plan, &qr, &kr, &vr, a.dim, a.mask_ptr(), a.scale, out.data_ptr(),
                                         nullptr, wp, need, stream.stream()));
    return {out, stats};
}

std::tuple<Tensor, Tensor, Tensor> attention_backward(const Tensor& grad, const Tensor& q, const Tensor& k, const Tensor& v,
                                                      const AttentionPlan& plan, const Tensor& key_mask, double scale,
                                                      const Tensor& out, const Tensor& stats) {
    const AttnArgs a = attention_args(q, k, v, plan, key_mask, scale);
    check_same(grad, q, "cross_attention", "its gradient");
    c10::OptionalDeviceGuard guard(q.device());
    const auto stream = c10::hip::getCurrentHIPStream(q.get_device());
    plan.used_on(stream);
    const Tensor g = with_unit_values(grad);
    Tensor dq = at::empty(q.sizes(), q.options());
    Tensor dk = at::empty(k.sizes(), k.options());
    Tensor dv = at::empty(v.sizes(), v.options());
    const size_t need = relm_mp_cross_attention_backward_workspace_size(&plan.plan, a.dim);
    const Tensor ws = bytes(need, q);
    const relm_mp_head_rows gr = head_rows(g), qr = head_rows(a.q), kr = head_rows(a.k), vr = head_rows(a.v);
    raise_if(relm_mp_cross_attention_backward_kept(a.dtype, &plan.plan, &gr, &qr, &kr, &vr, a.dim, a.mask_ptr(), a.scale,
                                                   out.const_data_ptr(), stats.const_data_ptr<float>(), dq.data_ptr(),
                                                   dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), need, stream.stream()));
    return {dq, dk, dv};
}

// Keeps the inputs, the output and each row's maximum and total; the backward computes the
// probabilities again.
struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const std::optional<Tensor>& key_mask, const c10::intrusive_ptr<AttentionPlan>& plan,
                          double scale) {
        const Tensor mask = key_mask.value_or(Tensor());
        const auto [out, stats] = attention_forward(q, k, v, *plan, mask, scale, true);
        ctx->save_for_backward({q, k, v, mask, out, stats});
        ctx->saved_data["plan"] = plan;
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        refuse_tangents({&grads[0]}, "cross_attention backward");
        const auto plan = ctx->saved_data["plan"].toCustomClass<AttentionPlan>();
        const auto [dq, dk, dv] = attention_backward(grads[0], s[0], s[1], s[2], *plan, s[3],
                                                     ctx->saved_data["scale"].toDouble(), s[4], s[5]);
        return once({dq, dk, dv, Tensor(), Tensor(), Tensor()}, "cross_attention");
    }
};

}  // namespace

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t plan, const std::optional<Tensor>& key_mask,
                       double scale) {
    refuse_tangents({&q, &k, &v}, "cross_attention");
    const auto p = plan_of(plan, "cross_attention");
    if (wants_grad({&q, &k, &v})) return CrossAttention::apply(q, k, v, key_mask, p, scale);
    return std::get<0>(attention_forward(q, k, v, *p, key_mask.value_or(Tensor()), scale, false));
}

// ---- orthogonalised update ---------------------------------------------------------

// One result per update; updates of more than two dimensions are stacks of matrices.
std::vector<Tensor> orthogonalise(at::TensorList updates, int64_t steps, at::ArrayRef<double> coefficients, double eps) {
    const char* op = "orthogonalise";
    TORCH_CHECK_VALUE(coefficients.size() == 3, op, ": three coefficients expected.");
    std::vector<Tensor> inputs, results;
    if (updates.empty()) return results;
    const int dtype = value_dtype(updates[0], op, "every update");
    std::vector<relm_mp_update> mats;
    c10::OptionalDeviceGuard guard(updates[0].device());
    inputs.reserve(updates.size());
    results.reserve(updates.size());
    mats.reserve(updates.size());
    for (const Tensor& u : updates) {
        refuse_tangents({&u}, op);
        check_like(u, updates[0], op, "every update");
        TORCH_CHECK_VALUE(u.dim() >= 2, op, ": updates must be matrices or stacks of them.");
        const int64_t rows = u.size(-2), cols = u.size(-1);
        const bool rows_apart = u.dim() == 2 && (cols <= 1 || u.stride(1) == 1) && (rows <= 1 || u.stride(0) >= cols);
        inputs.push_back(rows_apart ? u : u.contiguous());
        results.push_back(at::empty(u.sizes(), u.options()));
        const Tensor& in = inputs.back();
        const int64_t stride = u.dim() == 2 ? std::max(in.stride(0), cols) : cols;
        const int64_t step = rows * cols * static_cast<int64_t>(u.element_size());
        for (int64_t i = 0, n = step == 0 ? 0 : u.numel() / (rows * cols); i < n; ++i)
            mats.push_back({static_cast<const char*>(in.const_data_ptr()) + i * step,
                            static_cast<char*>(results.back().data_ptr()) + i * step, rows, cols, stride});
    }
    TORCH_CHECK(mats.size() <= 1 << 20, op, ": too many matrices.");
    const int32_t count = static_cast<int32_t>(mats.size());
    const size_t need = relm_mp_orthogonalise_workspace_size(mats.data(), count);
    const Tensor ws = need > 0 ? bytes(need, updates[0]) : Tensor();
    raise_if(relm_mp_orthogonalise(dtype, mats.data(), count, static_cast<int32_t>(std::clamp<int64_t>(steps, -1, 1 << 30)),
                                   static_cast<float>(coefficients[0]), static_cast<float>(coefficients[1]),
                                   static_cast<float>(coefficients[2]), static_cast<float>(eps),
                                   need > 0 ? ws.data_ptr() : nullptr, need, current_stream(updates[0])));
    return results;
}

}  // namespace readout
}  // namespace relm_amd

TORCH_LIBRARY_FRAGMENT(relm_mp, m) {
    m.def("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor)");
    m.def("rms_norm(Tensor x, Tensor weight, float eps) -> Tensor");
    m.def("add_rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
    m.class_<relm_amd::readout::AttentionPlan>("AttentionPlan");
    m.def("attention_plan(Tensor q_offsets, Tensor k_offsets, int heads, int kv_heads) -> (__torch__.torch.classes.relm_mp.AttentionPlan, int, Tensor)");
    m.def("cross_attention(Tensor q, Tensor k, Tensor v, int plan, Tensor? key_mask, float scale) -> Tensor");
    m.def("orthogonalise(Tensor[] updates, int steps, float[] coefficients, float eps) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(relm_mp, CompositeImplicitAutograd, m) {
    m.impl("add_rms_norm", relm_amd::readout::add_rms_norm);
    m.impl("rms_norm", relm_amd::readout::rms_norm);
    m.impl("add_rms_norm_fp8", relm_amd::readout::add_rms_norm_fp8);
    m.impl("attention_plan", relm_amd::readout::attention_plan);
    m.impl("cross_attention", relm_amd::readout::cross_attention);
    m.impl("orthogonalise", relm_amd::readout::orthogonalise);
}
