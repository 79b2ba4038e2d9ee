// C ABI of the readout ops (include/relm_mp.h): argument checks, then the kernels
// of norm_kernels.hip, attention_kernels.hip and orthogonal_kernels.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <exception>
#include <string>

#include "attention.h"
#include "internal.h"
#include "orthogonal.h"
#include "relm_mp.h"

namespace relm_mp {

namespace {

int bad(const std::string& what) { return set_error(RELM_MP_ERR_INVALID_ARGUMENT, "relm_mp " + what); }

bool value_dtype(int dtype) { return dtype == RELM_MP_F32 || dtype == RELM_MP_BF16 || dtype == RELM_MP_F16; }

#define RELM_TRY(expr)                     \
    do {                                   \
        const int _rc = (expr);            \
        if (_rc != RELM_MP_OK) return _rc; \
    } while (0)

#define RELM_HIP(expr, what)                              \
    do {                                                  \
        const hipError_t _e = (expr);                     \
        if (_e != hipSuccess) return hip_error(_e, what); \
    } while (0)

int check_workspace(const void* workspace, size_t bytes, size_t need, const char* op) {
    if (need == 0) return RELM_MP_OK;
    if (workspace == nullptr || bytes < need)
        return set_error(RELM_MP_ERR_WORKSPACE, std::string("relm_mp ") + op + ": workspace too small");
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return bad(std::string(op) + ": workspace not 16-byte aligned");
    return RELM_MP_OK;
}

int check_norm(int dtype, int64_t rows, int64_t width) {
    if (!value_dtype(dtype)) return bad("add_rms_norm: dtype must be f32, bf16 or f16");
    if (rows < 0 || rows > RELM_MP_MAX_ROWS) return bad("add_rms_norm: rows must be in [0, 2^31 - 2]");
    if (width < 0 || width > (1 << 24)) return bad("add_rms_norm: width must be in [0, 2^24]");
    return RELM_MP_OK;
}

int norm(int dtype, const void* x, const void* r, const void* w, int64_t rows, int64_t width, float eps, void* y, void* h,
         float* rstd, float* scale, bool fp8, relm_mp_stream_t stream) {
    RELM_TRY(check_norm(dtype, rows, width));
    if (!(eps >= 0.0f) || std::isinf(eps)) return bad("add_rms_norm: eps must be finite and not negative");
    if (rows == 0 || width == 0) return RELM_MP_OK;
    if (x == nullptr || w == nullptr || y == nullptr || (fp8 && scale == nullptr)) return bad("add_rms_norm: NULL array");
    RELM_HIP(launch_add_rms_norm(dtype, x, r, w, rows, width, eps, y, h, rstd, scale, static_cast<hipStream_t>(stream)),
             "relm_mp add_rms_norm kernel");
    return RELM_MP_OK;
}

// The backward's delta first, then the rows' statistics where only their lse is given, then the
// parts of dq or of dk and dv (one after the other in the same memory).
size_t delta_bytes(const relm_mp_attention_plan& p) {
    return align_up(static_cast<size_t>(p.q_rows) * p.heads * sizeof(float), 256);
}
size_t stats_bytes(const relm_mp_attention_plan& p) {
    return align_up(static_cast<size_t>(p.q_rows) * p.heads * sizeof(RowStats), 256);
}

bool null_rows(const relm_mp_head_rows* r) { return r == nullptr || r->data == nullptr; }

int check_attention(int dtype, const relm_mp_attention_plan* plan, int64_t head_dim, float scale) {
    if (plan == nullptr) return bad("cross_attention: NULL plan");
    if (!value_dtype(dtype)) return bad("cross_attention: dtype must be f32, bf16 or f16");
    if (head_dim < 1 || head_dim > RELM_MP_MAX_HEAD_DIM) return bad("cross_attention: head_dim must be in [1, 128]");
    if (!(scale > 0.0f) || std::isinf(scale)) return bad("cross_attention: scale must be finite and positive");
    if (plan->table == nullptr && plan->table_bytes > 0) return bad("cross_attention: the plan has no table");
    return RELM_MP_OK;
}

int attention_forward(int dtype, const relm_mp_attention_plan* plan, const relm_mp_head_rows* q, const relm_mp_head_rows* k,
                      const relm_mp_head_rows* v, int64_t head_dim, const uint8_t* key_mask, float scale, void* out, float* lse,
                      RowStats* stats, void* workspace, size_t workspace_bytes, relm_mp_stream_t stream) {
    RELM_TRY(check_attention(dtype, plan, head_dim, scale));
    if (plan->q_rows == 0) return RELM_MP_OK;
    if (null_rows(q) || out == nullptr || (plan->k_rows > 0 && (null_rows(k) || null_rows(v))))
        return bad("cross_attention: NULL array");
    RELM_TRY(check_workspace(workspace, workspace_bytes, relm_mp_cross_attention_workspace_size(plan, head_dim),
                             "cross_attention"));
    AttnOperands o{};
    o.q = *q;
    if (plan->k_rows > 0) {
        o.k = *k;
        o.v = *v;
    }
    o.head_dim = head_dim;
    o.key_mask = key_mask;
    o.scale = scale;
    o.out = out;
    o.lse = lse;
    o.stats = stats;
    o.parts = static_cast<float*>(workspace);
    RELM_HIP(launch_cross_attention(dtype, *plan, o, static_cast<hipStream_t>(stream)), "relm_mp cross_attention kernel");
    return RELM_MP_OK;
}

// From the rows' statistics, or from their lse (then stats is NULL).
int attention_backward(int dtype, const relm_mp_attention_plan* plan, const relm_mp_head_rows* grad, const relm_mp_head_rows* q,
                       const relm_mp_head_rows* k, const relm_mp_head_rows* v, int64_t head_dim, const uint8_t* key_mask,
                       float scale, const void* out, const float* lse, const RowStats* stats, void* dq, void* dk, void* dv,
                       void* workspace, size_t workspace_bytes, relm_mp_stream_t stream) {
    RELM_TRY(check_attention(dtype, plan, head_dim, scale));
    if (plan->q_rows == 0 && plan->k_rows == 0) return RELM_MP_OK;
    if ((plan->q_rows > 0 &&
         (null_rows(grad) || null_rows(q) || out == nullptr || (lse == nullptr && stats == nullptr) || dq == nullptr)) ||
        (plan->k_rows > 0 && (null_rows(k) || null_rows(v) || dk == nullptr || dv == nullptr)))
        return bad("cross_attention_backward: NULL array");
    RELM_TRY(check_workspace(workspace, workspace_bytes, relm_mp_cross_attention_backward_workspace_size(plan, head_dim),
                             "cross_attention_backward"));
    char* const at = static_cast<char*>(workspace);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    AttnOperands o{};
    if (plan->q_rows > 0) {
        o.q = *q;
        o.grad = *grad;
    }
    if (plan->k_rows > 0) {
        o.k = *k;
        o.v = *v;
    }
    o.head_dim = head_dim;
    o.key_mask = key_mask;
    o.scale = scale;
    o.out = const_cast<void*>(out);  // read only
    o.delta = reinterpret_cast<float*>(at);
    o.stats = const_cast<RowStats*>(stats);
    if (stats == nullptr) {
        o.stats = reinterpret_cast<RowStats*>(at + delta_bytes(*plan));
        RELM_HIP(launch_attention_stats(*plan, lse, scale, o.stats, st), "relm_mp cross_attention statistics kernel");
    }
    o.dq = dq;
    o.dk = dk;
    o.dv = dv;
    o.parts = reinterpret_cast<float*>(at + delta_bytes(*plan) + stats_bytes(*plan));
    RELM_HIP(launch_cross_attention_backward(dtype, *plan, o, st), "relm_mp cross_attention backward kernels");
    return RELM_MP_OK;
}

// The rule of a polynomial, with the scales that its values need; an error where the
// iteration leaves [-2, 2] (seen on a grid of starting values).
int ortho_rule(int32_t steps, float a, float b, float c, float eps, OrthoRule* rule) {
    if (steps < 1 || steps > RELM_MP_MAX_ORTHO_STEPS) return bad("orthogonalise: steps must be in [1, 64]");
    if (!(eps >= 0.0f) || std::isinf(eps)) return bad("orthogonalise: eps must be finite and not negative");
    double most_b = 1e-3;
    for (int i = 0; i <= 1024; ++i) {
        double x = i / 1024.0;
        for (int32_t s = 0; s < steps; ++s) {
            const double factor = b * x * x + c * x * x * x * x;
            most_b = std::max(most_b, std::fabs(factor));
            x = (a + factor) * x;
            if (!(std::fabs(x) <= 2.0))
                return bad("orthogonalise: these coefficients take singular values past 2");
        }
    }
    *rule = OrthoRule{a, b, c, eps, 4096.0f, std::ldexp(1.0f, std::max(-10, std::min(13, std::ilogb(30000.0 / most_b)))), steps};
    return RELM_MP_OK;
}

int check_updates(const relm_mp_update* updates, int32_t count) {
    if (count < 0 || (count > 0 && updates == nullptr)) return bad("orthogonalise: NULL or negative argument");
    for (int32_t i = 0; i < count; ++i) {
        const relm_mp_update& u = updates[i];
        if (u.rows < 0 || u.cols < 0 || u.rows > RELM_MP_MAX_ORTHO_SIDE || u.cols > RELM_MP_MAX_ORTHO_SIDE)
            return bad("orthogonalise: rows and columns must be in [0, 65536]");
        if (u.rows == 0 || u.cols == 0) continue;
        if (u.in == nullptr || u.out == nullptr) return bad("orthogonalise: NULL array");
        if (u.rows > 1 && u.row_stride < u.cols) return bad("orthogonalise: rows overlap");
    }
    return RELM_MP_OK;
}

}  // namespace

}  // namespace relm_mp

using namespace relm_mp;

extern "C" {

int relm_mp_add_rms_norm(int dtype, const void* x, const void* r, const void* w, int64_t rows, int64_t width, float eps,
                         void* y, void* h, float* rstd, relm_mp_stream_t stream) {
    return norm(dtype, x, r, w, rows, width, eps, y, h, rstd, nullptr, false, stream);
}

int relm_mp_add_rms_norm_fp8(int dtype, const void* x, const void* r, const void* w, int64_t rows, int64_t width, float eps,
                             void* q, float* scale, void* h, relm_mp_stream_t stream) {
    return norm(dtype, x, r, w, rows, width, eps, q, h, nullptr, scale, true, stream);
}

size_t relm_mp_add_rms_norm_backward_workspace_size(int dtype, int64_t rows, int64_t width) {
    return value_dtype(dtype) ? add_rms_norm_backward_workspace(dtype, rows, width) : 0;
}

int relm_mp_add_rms_norm_backward(int dtype, const void* dy, const void* dh, const void* h, const void* w, const float* rstd,
                                  int64_t rows, int64_t width, void* dx, void* dw, void* workspace, size_t workspace_bytes,
                                  relm_mp_stream_t stream) {
    RELM_TRY(check_norm(dtype, rows, width));
    if (width == 0) return RELM_MP_OK;
    RELM_TRY(check_workspace(workspace, workspace_bytes, add_rms_norm_backward_workspace(dtype, rows, width),
                             "add_rms_norm_backward"));
    if (dw == nullptr || (rows > 0 && (dy == nullptr || h == nullptr || w == nullptr || rstd == nullptr || dx == nullptr)))
        return bad("add_rms_norm_backward: NULL array");
    RELM_HIP(launch_add_rms_norm_backward(dtype, dy, dh, h, w, rstd, rows, width, dx, dw, static_cast<float*>(workspace),
                                          static_cast<hipStream_t>(stream)),
             "relm_mp add_rms_norm backward kernels");
    return RELM_MP_OK;
}

int relm_mp_attention_plan_build(const int64_t* q_offsets, const int64_t* k_offsets, int64_t graphs, int64_t q_rows,
                                 int64_t k_rows, int32_t heads, int32_t kv_heads, void* table, size_t table_bytes,
                                 relm_mp_attention_plan* plan) {
    try {
        return build_attention_plan(q_offsets, k_offsets, graphs, q_rows, k_rows, heads, kv_heads, table, table_bytes, plan);
    } catch (const std::exception& e) {  // host memory
        return bad(std::string("attention plan: ") + e.what());
    }
}

size_t relm_mp_cross_attention_workspace_size(const relm_mp_attention_plan* plan, int64_t head_dim) {
    return plan == nullptr ? 0 : attention_part_floats(*plan, head_dim) * sizeof(float);
}

int relm_mp_cross_attention(int dtype, const relm_mp_attention_plan* plan, const relm_mp_head_rows* q,
                            const relm_mp_head_rows* k, const relm_mp_head_rows* v, int64_t head_dim, const uint8_t* key_mask,
                            float scale, void* out, float* lse, void* workspace, size_t workspace_bytes,
                            relm_mp_stream_t stream) {
    return attention_forward(dtype, plan, q, k, v, head_dim, key_mask, scale, out, lse, nullptr, workspace, workspace_bytes,
                             stream);
}

int relm_mp_cross_attention_keep(int dtype, const relm_mp_attention_plan* plan, const relm_mp_head_rows* q,
                                 const relm_mp_head_rows* k, const relm_mp_head_rows* v, int64_t head_dim,
                                 const uint8_t* key_mask, float scale, void* out, float* stats, void* workspace,
                                 size_t workspace_bytes, relm_mp_stream_t stream) {
    if (plan != nullptr && plan->q_rows > 0 && stats == nullptr) return bad("cross_attention_keep: NULL array");
    return attention_forward(dtype, plan, q, k, v, head_dim, key_mask, scale, out, nullptr, reinterpret_cast<RowStats*>(stats),
                             workspace, workspace_bytes, stream);
}

size_t relm_mp_cross_attention_backward_workspace_size(const relm_mp_attention_plan* plan, int64_t head_dim) {
    if (plan == nullptr) return 0;
    return delta_bytes(*plan) + stats_bytes(*plan) +
           std::max(attention_part_floats(*plan, head_dim), attention_key_part_floats(*plan, head_dim)) * sizeof(float);
}

int relm_mp_cross_attention_backward(int dtype, const relm_mp_attention_plan* plan, const relm_mp_head_rows* grad,
                                     const relm_mp_head_rows* q, const relm_mp_head_rows* k, const relm_mp_head_rows* v,
                                     int64_t head_dim, const uint8_t* key_mask, float scale, const void* out, const float* lse,
                                     void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                     relm_mp_stream_t stream) {
    return attention_backward(dtype, plan, grad, q, k, v, head_dim, key_mask, scale, out, lse, nullptr, dq, dk, dv, workspace,
                              workspace_bytes, stream);
}

int relm_mp_cross_attention_backward_kept(int dtype, const relm_mp_attention_plan* plan, const relm_mp_head_rows* grad,
                                          const relm_mp_head_rows* q, const relm_mp_head_rows* k, const relm_mp_head_rows* v,
                                          int64_t head_dim, const uint8_t* key_mask, float scale, const void* out,
                                          const float* stats, void* dq, void* dk, void* dv, void* workspace,
                                          size_t workspace_bytes, relm_mp_stream_t stream) {
    return attention_backward(dtype, plan, grad, q, k, v, head_dim, key_mask, scale, out, nullptr,
                              reinterpret_cast<const RowStats*>(stats), dq, dk, dv, workspace, workspace_bytes, stream);
}

size_t relm_mp_orthogonalise_workspace_size(const relm_mp_update* updates, int32_t count) {
    if (check_updates(updates, count) != RELM_MP_OK) return 0;
    return orthogonalise_workspace(updates, count);
}

int relm_mp_orthogonalise(int dtype, const relm_mp_update* updates, int32_t count, int32_t steps, float a, float b, float c,
                          float eps, void* workspace, size_t workspace_bytes, relm_mp_stream_t stream) {
    if (!value_dtype(dtype)) return bad("orthogonalise: dtype must be f32, bf16 or f16");
    OrthoRule rule;
    RELM_TRY(ortho_rule(steps, a, b, c, eps, &rule));
    RELM_TRY(check_updates(updates, count));
    RELM_TRY(check_workspace(workspace, workspace_bytes, orthogonalise_workspace(updates, count), "orthogonalise"));
    try {
        RELM_HIP(launch_orthogonalise(dtype, updates, count, rule, workspace, static_cast<hipStream_t>(stream)),
                 "relm_mp orthogonalise kernels");
    } catch (const std::exception& e) {  // host memory
        return bad(std::string("orthogonalise: ") + e.what());
    }
    return RELM_MP_OK;
}

}  // extern "C"
