// C ABI of the norms and 8-bit products (include/dsa_mi355x_layer.h): argument
// checks and launches.  Like abi.cpp it never throws and never allocates.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/dsa_mi355x_layer.h"
#include "host_entry.h"
#include "kernels.h"

namespace {

int fail(int code, const char* fmt, ...) {
    char text[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    return dsa::set_error(code, "%s", text);
}

int finish(int rc, const char* what) {
    if (rc) return fail(rc, "%s: %s (hipError_t %d)", what, hipGetErrorString((hipError_t)rc), rc);
    return dsa::set_error(0, "%s", "");
}

bool aligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

bool known(int dtype) { return dtype == DSA_BF16 || dtype == DSA_F16 || dtype == DSA_F32; }

int check_rows(int64_t rows, int dim, int dtype, int64_t stride, int64_t other) {
    if (!known(dtype)) return fail(-1, "unknown dtype %d", dtype);
    if (dim <= 0 || dim > DSA_NORM_MAX_DIM)
        return fail(-1, "dim must be in [1, %d] (got %d)", DSA_NORM_MAX_DIM, dim);
    if (rows <= 0 || rows > (int64_t)1 << 40) return fail(-1, "rows must be in [1, 2^40]");
    if (stride < 0 || other < 0 || stride > (int64_t)1 << 40 || other > (int64_t)1 << 40 ||
        (stride > 0 && rows > ((int64_t)1 << 61) / stride) || (other > 0 && rows > ((int64_t)1 << 61) / other))
        return fail(-1, "strides must be in [0, 2^40], and rows * stride at most 2^61");
    return 0;
}

int check_norm(const dsa_norm_args* a, bool codes) {
    if (!a || !a->x || !a->out || (!codes && !a->weight) || (codes && !a->scales) || (a->residual && !a->sum))
        return fail(-1, "NULL pointer argument");
    if (const int rc = check_rows(a->rows, a->dim, a->dtype, a->x_stride, a->residual ? a->residual_stride : 0)) return rc;
    if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(-1, "eps must be a finite number, not negative");
    if (codes && (a->dim % 16 || !aligned(a->out, 16)))
        return fail(-1, "codes need dim a multiple of 16 (got %d) and a 16-byte aligned out", a->dim);
    if (codes && a->residual && !a->weight) return fail(-1, "a residual goes with a norm's weight");
    const unsigned size = a->dtype == DSA_F32 ? 4 : 2;
    if (!aligned(a->x, size) || !aligned(a->residual, size) || !aligned(a->out, codes ? 1 : size) || !aligned(a->sum, size) ||
        !aligned(a->weight, a->weight_f32 ? 4 : size) || !aligned(a->scales, 4) || !aligned(a->inverse, 4))
        return fail(-1, "pointers must be aligned to their elements");
    return 0;
}

// Whether all rows can be read and written 16 bytes at a time.
bool norm_vector(const dsa_norm_args* a, bool codes) {
    const int64_t step = a->dtype == DSA_F32 ? 4 : 8;
    return a->dim % 8 == 0 && aligned(a->x, 16) && a->x_stride % step == 0 && aligned(a->weight, 16) &&
           (codes || aligned(a->out, 16)) &&
           (!a->residual || (aligned(a->residual, 16) && a->residual_stride % step == 0 && aligned(a->sum, 16)));
}

int check_product(const dsa_product_args* a) {
    if (!a) return fail(-1, "args is NULL");
    if (a->M <= 0 || a->N <= 0 || a->K <= 0) return fail(-1, "M, N, K must be positive (got %d, %d, %d)", a->M, a->N, a->K);
    if (a->K % 16 || a->K >= 1 << 20) return fail(-1, "K must be a multiple of 16 below 2^20 (got %d)", a->K);
    if (a->M > 1 << 24 || a->N > 1 << 24) return fail(-1, "M and N must be at most 2^24 (got %d, %d)", a->M, a->N);
    if ((int64_t)a->M * a->N > (int64_t)1 << 37) return fail(-1, "M * N must be at most 2^37 (got %d, %d)", a->M, a->N);
    if (!known(a->dtype)) return fail(-1, "unknown dtype %d", a->dtype);
    return 0;
}

}  // namespace

extern "C" {

int dsa_rms_norm(const dsa_norm_args* a, void* stream) {
    if (const int rc = check_norm(a, false)) return rc;
    return finish(dsa::launch_norm(*a, false, norm_vector(a, false), static_cast<hipStream_t>(stream)), "norm launch");
}

int dsa_rms_norm_fp8(const dsa_norm_args* a, void* stream) {
    if (const int rc = check_norm(a, true)) return rc;
    return finish(dsa::launch_norm(*a, true, norm_vector(a, true), static_cast<hipStream_t>(stream)), "norm launch");
}

int64_t dsa_rms_norm_grad_ws_bytes(int64_t rows, int dim) {
    if (const int rc = check_rows(rows, dim, DSA_F32, 0, 0)) return rc;
    dsa::set_error(0, "%s", "");
    return dsa::norm_grad_teams(rows, dim) * dim * 4;
}

int dsa_rms_norm_grad(const dsa_norm_grad_args* a, void* stream) {
    if (!a || !a->h || !a->inverse || !a->weight || !a->grad_out || !a->grad_in || (a->grad_weight && !a->workspace))
        return fail(-1, "NULL pointer argument");
    if (const int rc = check_rows(a->rows, a->dim, a->dtype, a->h_stride, 0)) return rc;
    const unsigned size = a->dtype == DSA_F32 ? 4 : 2, wide = a->weight_f32 ? 4 : size;
    if (!aligned(a->h, size) || !aligned(a->grad_out, size) || !aligned(a->grad_sum, size) || !aligned(a->grad_in, size) ||
        !aligned(a->weight, wide) || !aligned(a->grad_weight, wide) || !aligned(a->inverse, 4) || !aligned(a->workspace, 16))
        return fail(-1, "pointers must be aligned to their elements, the workspace to 16 bytes");
    if (a->grad_weight) {
        const int64_t need = dsa::norm_grad_teams(a->rows, a->dim) * a->dim * 4;
        if (a->workspace_bytes < need)
            return fail(-1, "workspace of %lld bytes is below the %lld needed", (long long)a->workspace_bytes,
                        (long long)need);
    }
    const int64_t step = a->dtype == DSA_F32 ? 4 : 8;
    const bool vector = a->dim % 8 == 0 && aligned(a->h, 16) && a->h_stride % step == 0 && aligned(a->weight, 16) &&
                        aligned(a->grad_out, 16) && aligned(a->grad_sum, 16) && aligned(a->grad_in, 16);
    return finish(dsa::launch_norm_grad(*a, vector, static_cast<hipStream_t>(stream)), "norm gradient launch");
}

int dsa_matmul_fp8(const dsa_product_args* a, void* stream) {
    if (const int rc = check_product(a)) return rc;
    if (!a->a || !a->a_scales || !a->b || !a->b_scales || !a->out)
        return fail(-1, "NULL pointer argument");
    if (!aligned(a->a, 16) || !aligned(a->b, 16) || !aligned(a->a_scales, 4) || !aligned(a->b_scales, 4) ||
        !aligned(a->out, a->dtype == DSA_F32 ? 4 : 2))
        return fail(-1, "codes must be 16-byte aligned, scales and out to their elements");
    int device = 0, cus = 0;
    int rc = (int)hipGetDevice(&device);
    if (!rc) rc = (int)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
    if (rc) return fail(rc, "device query: %s", hipGetErrorString((hipError_t)rc));
    return finish(dsa::launch_product(*a, cus, static_cast<hipStream_t>(stream)), "product launch");
}

int dsa_product_tile(int M, int N, int K, int dtype, int cus) {
    dsa_product_args a{};
    a.M = M;
    a.N = N;
    a.K = K;
    a.dtype = dtype;
    if (const int rc = check_product(&a)) return rc;
    if (cus <= 0 || cus > 1 << 16) return fail(-1, "cus must be in [1, 2^16] (got %d)", cus);
    dsa::set_error(0, "%s", "");
    return dsa::product_tile(a, cus);
}

unsigned dsa_product_tiles(int dtype) { return known(dtype) ? dsa::product_tiles(dtype) : 0; }

}  // extern "C"
