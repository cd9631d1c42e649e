// Host fast path of dsa_amd.rms_norm, rms_norm_fp8, quantize_fp8 and matmul_fp8 (no
// reference counterpart: the reference takes q and kv as given, README.md:19-21).
//
// As fast_cache.cpp: a decode step's kernels take less time than their checks in
// Python.  Nothing is raised for a bad input: whatever the Python path would reject,
// and what it does besides (a gradient to record, nothing to do), returns None, and
// the caller goes on in Python.  A failed launch returns the library's status code.
// Nothing is allocated or launched before every check has passed.
#include <cmath>
#include <cstdint>

#include "dsa_mi355x_layer.h"
#include "fast_args.h"

namespace {

decltype(&dsa_rms_norm) g_norm = nullptr;
decltype(&dsa_rms_norm_fp8) g_norm_fp8 = nullptr;
decltype(&dsa_matmul_fp8_ws_bytes) g_product_bytes = nullptr;
decltype(&dsa_matmul_fp8) g_product = nullptr;

int code_of(at::ScalarType type) {
    return type == at::kBFloat16 ? DSA_BF16 : type == at::kHalf ? DSA_F16 : type == at::kFloat ? DSA_F32 : -1;
}

// Elements between rows of the last dimension; false where they are not evenly spaced or not contiguous themselves.
bool row_stride(const at::Tensor& t, int64_t& stride) {
    const int64_t n = t.dim();
    if (t.size(n - 1) > 1 && t.stride(n - 1) != 1) return false;
    stride = t.size(n - 1);
    int64_t next = -1;  // what the next dimension's stride has to be
    for (int64_t i = n - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (next < 0) stride = t.stride(i);
        else if (t.stride(i) != next) return false;
        next = t.stride(i) * t.size(i);
    }
    return true;
}

bool recorded(const at::Tensor* t) { return t && ((at::GradMode::is_enabled() && t->requires_grad()) || differentiated(*t)); }

// Without a weight: codes of x itself.
py::object norm(py::handle hx, const at::Tensor* weight, const at::Tensor* residual, double eps, bool codes, bool pow2) {
    const at::Tensor* x = tensor(hx);
    if (!x || x->dim() < 1 || x->numel() == 0) return py::none();
    const c10::Device dev = x->device();
    const auto type = x->scalar_type();
    const int64_t dim = x->size(-1);
    dsa_norm_args a{};
    a.dtype = code_of(type);
    if (!dev.is_cuda() || a.dtype < 0 || dim > DSA_NORM_MAX_DIM || (codes && dim % 16) ||
        !(eps >= 0.0 && eps <= 3.4028234663852886e38) || !row_stride(*x, a.x_stride) || recorded(x))
        return py::none();
    if (weight) {
        if (weight->dim() != 1 || weight->size(0) != dim || weight->device() != dev || !weight->is_contiguous() ||
            (weight->scalar_type() != type && weight->scalar_type() != at::kFloat) || recorded(weight))
            return py::none();
        a.weight = weight->data_ptr();
        a.weight_f32 = weight->scalar_type() == at::kFloat;
    }
    if (residual) {
        if (residual->sizes() != x->sizes() || residual->scalar_type() != type || residual->device() != dev ||
            !row_stride(*residual, a.residual_stride) || recorded(residual))
            return py::none();
        a.residual = residual->data_ptr();
    }
    c10::DeviceGuard guard(dev);
    const auto options = x->options().requires_grad(false).memory_format(c10::nullopt);
    at::Tensor out = at::empty(x->sizes(), codes ? options.dtype(at::kFloat8_e4m3fn) : options), sum, scales;
    if (residual) {
        sum = at::empty(x->sizes(), options);
        a.sum = sum.data_ptr();
    }
    if (codes) {
        auto shape = x->sizes().vec();
        shape.back() = (dim + 127) / 128;
        scales = at::empty(shape, options.dtype(at::kFloat));
        a.scales = static_cast<float*>(scales.data_ptr());
        a.pow2_scales = pow2;
    }
    a.x = x->data_ptr();
    a.out = out.data_ptr();
    a.rows = x->numel() / dim;
    a.dim = (int32_t)dim;
    a.eps = (float)eps;
    auto* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    const int rc = codes ? g_norm_fp8(&a, stream) : g_norm(&a, stream);
    if (rc != 0) return py::int_(rc);
    if (codes) return residual ? py::object(py::make_tuple(out, scales, sum)) : py::object(py::make_tuple(out, scales));
    return residual ? py::object(py::make_tuple(out, sum)) : py::cast(out);
}

py::object with_weight(py::handle hx, py::handle hweight, py::handle hresidual, py::handle heps, bool codes, bool pow2) {
    const at::Tensor *weight = tensor(hweight), *residual = tensor(hresidual);
    if (!weight || (!residual && !hresidual.is_none()) || !PyFloat_CheckExact(heps.ptr())) return py::none();
    return norm(hx, weight, residual, PyFloat_AS_DOUBLE(heps.ptr()), codes, pow2);
}

py::object rms_norm(py::handle hx, py::handle hweight, py::handle hresidual, py::handle heps) {
    return with_weight(hx, hweight, hresidual, heps, false, false);
}

py::object rms_norm_fp8(py::handle hx, py::handle hweight, py::handle hresidual, py::handle heps, py::handle hpow2) {
    bool pow2;
    if (!flag(hpow2, pow2)) return py::none();
    return with_weight(hx, hweight, hresidual, heps, true, pow2);
}

py::object quantize_fp8(py::handle hx, py::handle hpow2) {
    bool pow2;
    if (!flag(hpow2, pow2)) return py::none();
    return norm(hx, nullptr, nullptr, 0.0, true, pow2);
}

py::object matmul_fp8(py::handle ha, py::handle ha_scales, py::handle hb, py::handle hb_scales, py::handle hdtype) {
    const at::Tensor *a = tensor(ha), *a_scales = tensor(ha_scales), *b = tensor(hb), *b_scales = tensor(hb_scales);
    if (!a || !a_scales || !b || !b_scales || a->dim() < 1 || b->dim() != 2 || a->numel() == 0 ||
        !THPDtype_Check(hdtype.ptr()))
        return py::none();
    const auto type = reinterpret_cast<THPDtype*>(hdtype.ptr())->scalar_type;
    const c10::Device dev = a->device();
    const int64_t N = b->size(0), K = b->size(1), blocks = (K + 127) / 128;
    dsa_product_args p{};
    p.dtype = code_of(type);
    if (!dev.is_cuda() || p.dtype < 0 || K <= 0 || K % 16 || K >= 1 << 20 || N <= 0 || N > 1 << 24 || a->size(-1) != K ||
        a->numel() / K > 1 << 24 || a_scales->dim() != a->dim() || a_scales->size(-1) != blocks ||
        a_scales->sizes().slice(0, a->dim() - 1) != a->sizes().slice(0, a->dim() - 1) ||
        !dims(*b_scales, {(N + 127) / 128, blocks}) || a->scalar_type() != at::kFloat8_e4m3fn ||
        b->scalar_type() != at::kFloat8_e4m3fn || a_scales->scalar_type() != at::kFloat ||
        b_scales->scalar_type() != at::kFloat)
        return py::none();
    for (const at::Tensor* t : {a, a_scales, b, b_scales})
        if (t->device() != dev || !t->is_contiguous() || !t->has_storage()) return py::none();
    p.a = static_cast<const uint8_t*>(a->data_ptr());
    p.a_scales = static_cast<const float*>(a_scales->data_ptr());
    p.b = static_cast<const uint8_t*>(b->data_ptr());
    p.b_scales = static_cast<const float*>(b_scales->data_ptr());
    if (!aligned(p.a, 16) || !aligned(p.b, 16)) return py::none();
    p.M = (int32_t)(a->numel() / K);
    p.N = (int32_t)N;
    p.K = (int32_t)K;
    c10::DeviceGuard guard(dev);
    p.workspace_bytes = g_product_bytes(&p);
    if (p.workspace_bytes < 0) return py::none();
    auto shape = a->sizes().vec();
    shape.back() = N;
    const auto options = a->options().requires_grad(false).memory_format(c10::nullopt);
    at::Tensor out = at::empty(shape, options.dtype(type)), workspace;
    if (p.workspace_bytes > 0) {
        workspace = at::empty({p.workspace_bytes}, options.dtype(at::kByte));
        p.workspace = workspace.data_ptr();
    }
    p.out = out.data_ptr();
    const int rc = g_product(&p, c10::hip::getCurrentHIPStream(dev.index()).stream());
    if (rc != 0) return py::int_(rc);
    return py::cast(out);
}

void set_entry(uint64_t norm_address, uint64_t norm_fp8, uint64_t product_bytes, uint64_t product) {
    g_norm = reinterpret_cast<decltype(g_norm)>(norm_address);
    g_norm_fp8 = reinterpret_cast<decltype(g_norm_fp8)>(norm_fp8);
    g_product_bytes = reinterpret_cast<decltype(g_product_bytes)>(product_bytes);
    g_product = reinterpret_cast<decltype(g_product)>(product);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("rms_norm", &rms_norm, "dsa_amd.rms_norm, or None");
    m.def("rms_norm_fp8", &rms_norm_fp8, "dsa_amd.rms_norm_fp8, or None");
    m.def("quantize_fp8", &quantize_fp8, "dsa_amd.quantize_fp8, or None");
    m.def("matmul_fp8", &matmul_fp8, "dsa_amd.matmul_fp8, or None");
    m.def("set_entry", &set_entry, "addresses of the library's entry points");
}
