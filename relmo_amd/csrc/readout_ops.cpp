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

}  // namespace readout
}  // namespace relm_amd

TORCH_LIBRARY_FRAGMENT(relm_mp, m) {
    m.def("add_rms_norm(Tensor x, Tensor? residual, Tensor weight, float eps, bool keep) -> (Tensor, Tensor, Tensor)");
    m.def("add_rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("add_rms_norm_backward(Tensor grad_y, Tensor? grad_h, Tensor h, Tensor weight, Tensor rstd) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(relm_mp, CompositeImplicitAutograd, m) {
    m.impl("add_rms_norm", relm_amd::readout::add_rms_norm);
    m.impl("add_rms_norm_fp8", relm_amd::readout::add_rms_norm_fp8);
    m.impl("add_rms_norm_backward", relm_amd::readout::add_rms_norm_backward);
}
