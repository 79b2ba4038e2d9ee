// C ABI of the readout ops (include/relm_mp.h): argument checks, then the kernels
// of norm_kernels.hip.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <string>

#include "internal.h"
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

}  // extern "C"
