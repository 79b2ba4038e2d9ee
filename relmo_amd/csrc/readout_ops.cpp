// Torch binding of the readout ops (the relm_mp namespace's second part; the
// message-passing ops are in relm_mp_ops.cpp).  No reference counterpart: what a
// program runs on the object states that the message passing leaves.  GPU tensors
// of float32, bfloat16 or float16; the facade runs ATen formulations for CPU
// tensors and holds the autograd functions.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <tuple>
#include <vector>

#include "relm_mp.h"

namespace relm_amd {
namespace readout {

using at::Tensor;

namespace {

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
    TORCH_CHECK(t.scalar_type() == like.scalar_type() && t.device() == like.device(), op, ": ", name,
                " must have the dtype and device of the first argument.");
}

void check_same(const Tensor& t, const Tensor& like, const char* op, const char* name) {
    check_like(t, like, op, name);
    TORCH_CHECK(t.sizes() == like.sizes(), op, ": ", name, " must have the shape of the first argument.");
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
    TORCH_CHECK(x.dim() >= 1, op, ": x must have at least one dimension.");
    a.width = x.size(-1);
    a.rows = a.width == 0 ? 0 : x.numel() / a.width;
    check_like(weight, x, op, "weight");
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == a.width, op, ": weight must be [", a.width, "].");
    if (residual.has_value() && residual->defined()) {
        check_same(*residual, x, op, "residual");
        a.r = residual->contiguous();
    }
    return a;
}

}  // namespace

// (y, h, rstd): h is empty without a residual (it would be x), rstd unless `keep`.
std::tuple<Tensor, Tensor, Tensor> add_rms_norm(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight,
                                                double eps, bool keep) {
    const NormArgs a = norm_args(x, residual, weight, "add_rms_norm");
    c10::OptionalDeviceGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), a.x.options());
    Tensor h = a.r.defined() ? at::empty(x.sizes(), a.x.options()) : at::empty({0}, a.x.options());
    Tensor rstd = at::empty({keep ? a.rows : 0}, a.x.options().dtype(at::kFloat));
    raise_if(relm_mp_add_rms_norm(a.dtype, a.x.const_data_ptr(), opt_ptr(a.r), a.w.const_data_ptr(), a.rows, a.width,
                                  static_cast<float>(eps), y.data_ptr(), a.r.defined() ? h.data_ptr() : nullptr,
                                  keep ? rstd.data_ptr<float>() : nullptr, current_stream(x)));
    return {y, h, rstd};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8(const Tensor& x, const std::optional<Tensor>& residual,
                                                    const Tensor& weight, double eps) {
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

std::tuple<Tensor, Tensor> add_rms_norm_backward(const Tensor& grad_y, const std::optional<Tensor>& grad_h, const Tensor& h,
                                                 const Tensor& weight, const Tensor& rstd) {
    const char* op = "add_rms_norm_backward";
    const NormArgs a = norm_args(h, std::nullopt, weight, op);
    check_same(grad_y, h, op, "grad_y");
    TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.device() == h.device() && rstd.numel() == a.rows, op,
                ": rstd must be the forward's, float32 [rows].");
    const Tensor gy = grad_y.contiguous(), rs = rstd.contiguous();
    Tensor gh;
    if (grad_h.has_value() && grad_h->defined()) {
        check_same(*grad_h, h, op, "grad_h");
        gh = grad_h->contiguous();
    }
    c10::OptionalDeviceGuard guard(h.device());
    Tensor dx = at::empty(h.sizes(), a.x.options());
    Tensor dw = at::empty(weight.sizes(), a.x.options());
    const size_t need = relm_mp_add_rms_norm_backward_workspace_size(a.dtype, a.rows, a.width);
    const Tensor ws = bytes(need, h);
    raise_if(relm_mp_add_rms_norm_backward(a.dtype, gy.const_data_ptr(), opt_ptr(gh), a.x.const_data_ptr(),
                                           a.w.const_data_ptr(), rs.const_data_ptr<float>(), a.rows, a.width, dx.data_ptr(),
                                           dw.data_ptr(), ws.data_ptr(), need, current_stream(h)));
    return {dx, dw};
}

// ---- cross attention -------------------------------------------------------------

// A batch's plan with its table on the device.  The table is copied there before the
// constructor returns, so any stream may use it; a stream other than the one the
// memory was allocated on is recorded with the allocator.
struct AttentionPlan : torch::CustomClassHolder {
    relm_mp_attention_plan plan{};
    Tensor table;
    hipStream_t stream = nullptr;

    void used_on(const c10::hip::HIPStream& s) const {
        if (table.numel() > 0 && s.stream() != stream)
            c10::hip::HIPCachingAllocator::recordStream(table.storage().data_ptr(), s);
    }
};

c10::intrusive_ptr<AttentionPlan> attention_plan(const Tensor& q_offsets, const Tensor& k_offsets, int64_t heads,
                                                 int64_t kv_heads) {
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
    const auto build = [&](void* table, size_t bytes) {
        raise_if(relm_mp_attention_plan_build(qo, ko, graphs, qo[graphs], ko[graphs], static_cast<int32_t>(heads),
                                              static_cast<int32_t>(kv_heads), table, bytes, &ref->plan));
    };
    build(nullptr, 0);
    Tensor table = at::empty({ref->plan.table_bytes}, at::kByte);
    if (ref->plan.table_bytes > 0) build(table.data_ptr(), static_cast<size_t>(ref->plan.table_bytes));
    const auto s = c10::hip::getCurrentHIPStream(q_offsets.get_device());
    ref->table = table.to(q_offsets.device());
    ref->stream = s.stream();
    ref->plan.table = ref->plan.table_bytes > 0 ? ref->table.const_data_ptr() : nullptr;
    return ref;
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

AttnArgs attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionPlan& p,
                        const std::optional<Tensor>& key_mask, double scale, const char* op) {
    AttnArgs a;
    a.dtype = value_dtype(q, op, "q");
    for (const Tensor* t : {&q, &k, &v}) {
        TORCH_CHECK(t->dim() == 3, op, ": q, k and v must be [rows, heads, head_dim].");
        check_like(*t, q, op, "k and v");
    }
    a.dim = q.size(2);
    TORCH_CHECK(a.dim >= 1 && a.dim <= RELM_MP_MAX_HEAD_DIM, op, ": head_dim must be in [1, ", RELM_MP_MAX_HEAD_DIM, "].");
    TORCH_CHECK(q.size(0) == p.plan.q_rows && q.size(1) == p.plan.heads, op, ": q must be [", p.plan.q_rows, ", ",
                p.plan.heads, ", head_dim] for this plan.");
    for (const Tensor* t : {&k, &v})
        TORCH_CHECK(t->size(0) == p.plan.k_rows && t->size(1) == p.plan.kv_heads && t->size(2) == a.dim, op,
                    ": k and v must be [", p.plan.k_rows, ", ", p.plan.kv_heads, ", ", a.dim, "] for this plan.");
    TORCH_CHECK(p.table.device() == q.device(), op, ": the plan is on another device.");
    a.q = with_unit_values(q);
    a.k = with_unit_values(k);
    a.v = with_unit_values(v);
    if (key_mask.has_value() && key_mask->defined()) {
        TORCH_CHECK(key_mask->dim() == 1 && key_mask->size(0) == p.plan.k_rows && key_mask->scalar_type() == at::kBool &&
                        key_mask->device() == q.device(),
                    op, ": key_mask must be bool [", p.plan.k_rows, "] on the device of q.");
        a.mask = key_mask->contiguous();
    }
    a.scale = static_cast<float>(scale);
    return a;
}

}  // namespace

// (out, lse); lse is empty unless `keep`.
std::tuple<Tensor, Tensor> cross_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                           const c10::intrusive_ptr<AttentionPlan>& plan,
                                           const std::optional<Tensor>& key_mask, double scale, bool keep) {
    const AttnArgs a = attention_args(q, k, v, *plan, key_mask, scale, "cross_attention");
    c10::OptionalDeviceGuard guard(q.device());
    plan->used_on(c10::hip::getCurrentHIPStream(q.get_device()));
    Tensor out = at::empty(q.sizes(), q.options());
    Tensor lse = keep ? at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))
                      : at::empty({0}, q.options().dtype(at::kFloat));
    const size_t need = relm_mp_cross_attention_workspace_size(&plan->plan, a.dim);
    const Tensor ws = need > 0 ? bytes(need, q) : Tensor();
    const relm_mp_head_rows qr = head_rows(a.q), kr = head_rows(a.k), vr = head_rows(a.v);
    raise_if(relm_mp_cross_attention(a.dtype, &plan->plan, &qr, &kr, &vr, a.dim, a.mask_ptr(), a.scale, out.data_ptr(),
                                     keep ? lse.data_ptr<float>() : nullptr, need > 0 ? ws.data_ptr() : nullptr, need,
                                     current_stream(q)));
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> cross_attention_backward(const Tensor& grad, const Tensor& q, const Tensor& k,
                                                            const Tensor& v, const c10::intrusive_ptr<AttentionPlan>& plan,
                                                            const std::optional<Tensor>& key_mask, double scale,
                                                            const Tensor& out, const Tensor& lse) {
    const char* op = "cross_attention_backward";
    const AttnArgs a = attention_args(q, k, v, *plan, key_mask, scale, op);
    check_same(grad, q, op, "grad");
    check_same(out, q, op, "out");
    TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.device() == q.device() && lse.dim() == 2 &&
                    lse.size(0) == q.size(0) && lse.size(1) == q.size(1),
                op, ": lse must be the forward's, float32 [rows, heads].");
    c10::OptionalDeviceGuard guard(q.device());
    plan->used_on(c10::hip::getCurrentHIPStream(q.get_device()));
    const Tensor g = with_unit_values(grad), o = out.contiguous(), l = lse.contiguous();
    Tensor dq = at::empty(q.sizes(), q.options());
    Tensor dk = at::empty(k.sizes(), k.options());
    Tensor dv = at::empty(v.sizes(), v.options());
    const size_t need = relm_mp_cross_attention_backward_workspace_size(&plan->plan, a.dim);
    const Tensor ws = bytes(need, q);
    const relm_mp_head_rows gr = head_rows(g), qr = head_rows(a.q), kr = head_rows(a.k), vr = head_rows(a.v);
    raise_if(relm_mp_cross_attention_backward(a.dtype, &plan->plan, &gr, &qr, &kr, &vr, a.dim, a.mask_ptr(), a.scale,
                                              o.const_data_ptr(), l.const_data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                                              dv.data_ptr(), ws.data_ptr(), need, current_stream(q)));
    return {dq, dk, dv};
}

// ---- orthogonalised update ---------------------------------------------------------

// One result per update; updates of more than two dimensions are stacks of matrices.
std::vector<Tensor> orthogonalise(at::TensorList updates, int64_t steps, at::ArrayRef<double> coefficients, double eps) {
    const char* op = "orthogonalise";
    TORCH_CHECK(coefficients.size() == 3, op, ": three coefficients expected.");
    std::vector<Tensor> inputs, results;
    if (updates.empty()) return results;
    const int dtype = value_dtype(updates[0], op, "every update");
    std::vector<relm_mp_update> mats;
    c10::OptionalDeviceGuard guard(updates[0].device());
    inputs.reserve(updates.size());
    results.reserve(updates.size());
    mats.reserve(updates.size());
    for (const Tensor& u : updates) {
        check_like(u, updates[0], op, "every update");
        TORCH_CHECK(u.dim() >= 2, op, ": updates must be matrices or stacks of them.");
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
    raise_if(relm_mp_orthogonalise(dtype, mats.data(), count, static_cast<int32_t>(std::min<int64_t>(steps, 1 << 30)),
                                   static_cast<float>(coefficients[0]), static_cast<float>(coefficients[1]),
                                   static_cast<float>(coefficients[2]), static_cast<float>(eps),
                                   need > 0 ? ws.data_ptr() : nullptr, need, current_stream(updates[0])));
    return results;
}

}  // namespace readout
}  // namespace relm_amd

TORCH_LIBRARY_FRAGMENT(relm_mp, m) {
    m.def("add_rms_norm(Tensor x, Tensor? residual, Tensor weight, float eps, bool keep) -> (Tensor, Tensor, Tensor)");
    m.def("add_rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("add_rms_norm_backward(Tensor grad_y, Tensor? grad_h, Tensor h, Tensor weight, Tensor rstd) -> (Tensor, Tensor)");
    m.class_<relm_amd::readout::AttentionPlan>("AttentionPlan");
    m.def("attention_plan(Tensor q_offsets, Tensor k_offsets, int heads, int kv_heads) -> __torch__.torch.classes.relm_mp.AttentionPlan");
    m.def("cross_attention(Tensor q, Tensor k, Tensor v, __torch__.torch.classes.relm_mp.AttentionPlan plan, Tensor? key_mask, float scale, bool keep) -> (Tensor, Tensor)");
    m.def("cross_attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, __torch__.torch.classes.relm_mp.AttentionPlan plan, Tensor? key_mask, float scale, Tensor out, Tensor lse) -> (Tensor, Tensor, Tensor)");
    m.def("orthogonalise(Tensor[] updates, int steps, float[] coefficients, float eps) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(relm_mp, CompositeImplicitAutograd, m) {
    m.impl("add_rms_norm", relm_amd::readout::add_rms_norm);
    m.impl("add_rms_norm_fp8", relm_amd::readout::add_rms_norm_fp8);
    m.impl("add_rms_norm_backward", relm_amd::readout::add_rms_norm_backward);
    m.impl("attention_plan", relm_amd::readout::attention_plan);
    m.impl("cross_attention", relm_amd::readout::cross_attention);
    m.impl("cross_attention_backward", relm_amd::readout::cross_attention_backward);
    m.impl("orthogonalise", relm_amd::readout::orthogonalise);
}
