// Host fast path of dsa_amd.rms_norm, rms_norm_fp8, quantize_fp8 and matmul_fp8 (no
// reference counterpart: the reference takes q and kv as given, README.md:19-21).
//
// As fast_cache.cpp: a decode step's kernels take less time than their checks in
// Python.  Nothing is raised for a bad input: whatever the Python path would reject,
// and what it does besides (nothing to do), returns None, and the caller goes on in
// Python.  A failed launch returns the library's status code, or raises where the
// gradient is recorded.  Nothing is allocated or launched before every check has passed.
//
// The norm's gradient is recorded here too: a training step's kernels took less time
// (4095 rows of 4096: 58 us) than a Python function's forward and backward (130).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdint>
#include <memory>
#include <optional>

#include "dsa_mi355x.h"
#include "dsa_mi355x_layer.h"
#include "fast_args.h"

namespace {

decltype(&dsa_rms_norm) g_norm = nullptr;
decltype(&dsa_rms_norm_fp8) g_norm_fp8 = nullptr;
decltype(&dsa_matmul_fp8) g_product = nullptr;
decltype(&dsa_rms_norm_grad_ws_bytes) g_grad_bytes = nullptr;
decltype(&dsa_rms_norm_grad) g_grad = nullptr;
decltype(&dsa_last_error) g_error = nullptr;

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

// Whether the fast path takes it: its memory holds its values as they are.
bool plain(const at::Tensor& t) { return !differentiated(t) && !t.is_neg(); }

bool wants_grad(const at::Tensor* t) { return t && at::GradMode::is_enabled() && t->requires_grad(); }

void* stream_of(c10::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, ": ", g_error()); }

// A tensor that was saved for the gradient.  Hooks of saved tensors may have put another
// in its place: equal, says their contract, but laid out in any way.
at::Tensor kept(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type, at::ScalarType other, c10::Device dev) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && (t.scalar_type() == type || t.scalar_type() == other) && t.device() == dev &&
                    t.layout() == at::kStrided,
                "rms_norm: a saved tensor came back with another shape, type or device");
    return t.is_neg() ? t.resolve_neg() : t;
}

// The norm with its gradient, of arguments that norm() has checked: as the function of
// the same name in dsa_amd/norm.py.
struct RmsNorm : torch::autograd::Function<RmsNorm> {
    using Context = torch::autograd::AutogradContext;
    using List = torch::autograd::variable_list;

    static List forward(Context* ctx, const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& residual,
                        double eps) {
        const c10::Device dev = x.device();
        dsa_norm_args a{};
        row_stride(x, a.x_stride);
        const auto options = x.options().requires_grad(false).memory_format(std::nullopt);
        at::Tensor y = at::empty(x.sizes(), options), h = x;
        at::Tensor inverse = at::empty(x.sizes().slice(0, x.dim() - 1), options.dtype(at::kFloat));
        if (residual) {
            row_stride(*residual, a.residual_stride);
            h = at::empty(x.sizes(), options);
            a.residual = residual->data_ptr();
            a.sum = h.data_ptr();
        }
        a.x = x.data_ptr();
        a.weight = weight.data_ptr();
        a.out = y.data_ptr();
        a.inverse = static_cast<float*>(inverse.data_ptr());
        a.dim = (int32_t)x.size(-1);
        a.rows = x.numel() / a.dim;
        a.dtype = code_of(x.scalar_type());
        a.weight_f32 = weight.scalar_type() == at::kFloat;
        a.eps = (float)eps;
        check(g_norm(&a, stream_of(dev)), "dsa_rms_norm");
        ctx->save_for_backward({h, weight, inverse});
        ctx->set_materialize_grads(false);
        return residual ? List{y, h} : List{y};
    }

    static List backward(Context* ctx, List grads) {
        at::Tensor grad_h, grad_weight;
        {
            at::NoGradGuard plain;
            const auto saved = ctx->get_saved_variables();
            // the node is called without any gradient too, where a function behind it gives none: of zeros then
            const at::Tensor& like = grads[0].defined() ? grads[0] : grads.size() > 1 && grads[1].defined() ? grads[1] : saved[0];
            const c10::Device dev = like.device();
            c10::DeviceGuard guard(dev);
            const auto type = like.scalar_type();
            at::Tensor h = kept(saved[0], like.sizes(), type, type, dev);
            const at::Tensor weight = kept(saved[1], like.sizes().slice(like.dim() - 1), type, at::kFloat, dev).contiguous();
            const at::Tensor inverse = kept(saved[2], like.sizes().slice(0, like.dim() - 1), at::kFloat, at::kFloat, dev).contiguous();
            const auto options = h.options().requires_grad(false).memory_format(std::nullopt);
            const at::Tensor grad_y = grads[0].defined() ? grads[0].resolve_neg().contiguous() : at::zeros(h.sizes(), options);
            at::Tensor grad_sum, workspace;
            grad_h = at::empty(h.sizes(), options);
            dsa_norm_grad_args a{};
            if (grads.size() > 1 && grads[1].defined()) {
                grad_sum = grads[1].resolve_neg().contiguous();
                a.grad_sum = grad_sum.data_ptr();
            }
            if (!row_stride(h, a.h_stride)) {
                h = h.contiguous();
                row_stride(h, a.h_stride);
            }
            a.h = h.data_ptr();
            a.inverse = static_cast<const float*>(inverse.data_ptr());
            a.weight = weight.data_ptr();
            a.grad_out = grad_y.data_ptr();
            a.grad_in = grad_h.data_ptr();
            a.dim = (int32_t)h.size(-1);
            a.rows = h.numel() / a.dim;
            a.dtype = code_of(h.scalar_type());
            a.weight_f32 = weight.scalar_type() == at::kFloat;
            if (ctx->needs_input_grad(1)) {
                grad_weight = at::empty(weight.sizes(), weight.options().requires_grad(false));
                a.workspace_bytes = g_grad_bytes(a.rows, a.dim);
                workspace = at::empty({a.workspace_bytes}, options.dtype(at::kByte));
                a.grad_weight = grad_weight.data_ptr();
                a.workspace = workspace.data_ptr();
            }
            check(g_grad(&a, stream_of(dev)), "dsa_rms_norm_grad");
        }
        List out{grad_h, grad_weight, grads.size() > 1 ? grad_h : at::Tensor(), at::Tensor()};
        if (at::GradMode::is_enabled()) {  // a graph of the gradients is built: there are none of the second order
            List some;
            for (const at::Tensor& t : out)
                if (t.defined()) some.push_back(t.detach().requires_grad_(true));
            const auto refuse = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)some.size());
            some = (*refuse)(std::move(some));
            size_t next = 0;
            for (at::Tensor& t : out)
                if (t.defined()) t = some[next++];
        }
        return out;
    }
};

// A leaf that some eager graph on the default stream still uses has its sums there, and
// a capture of the gradient, which runs on a stream of its own, would end in an error
// that no caller can catch.  Refused here, before anything of it is captured.
void check_capture(std::initializer_list<const at::Tensor*> leaves) {
    bool lives = false;
    for (const at::Tensor* t : leaves) {
        if (!wants_grad(t) || !t->is_leaf()) continue;
        const auto sums = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto stream = sums ? sums->stream() : std::nullopt;
        lives |= stream && stream->id() == 0;
    }
    if (!lives) return;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const int rc = (int)hipStreamIsCapturing(c10::hip::getCurrentHIPStream().stream(), &status);
    if (rc == 0 && status != hipStreamCaptureStatusNone)
        throw py::value_error("the gradient of a leaf cannot be captured while results that it was used for on the "
                              "default stream are kept: drop them first");
}

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
        !(eps >= 0.0 && eps <= 3.4028234663852886e38) || !row_stride(*x, a.x_stride) || !plain(*x))
        return py::none();
    if (weight) {
        if (weight->dim() != 1 || weight->size(0) != dim || weight->device() != dev || !weight->is_contiguous() ||
            (weight->scalar_type() != type && weight->scalar_type() != at::kFloat) || !plain(*weight))
            return py::none();
        a.weight = weight->data_ptr();
        a.weight_f32 = weight->scalar_type() == at::kFloat;
    }
    if (residual) {
        if (residual->sizes() != x->sizes() || residual->scalar_type() != type || residual->device() != dev ||
            !row_stride(*residual, a.residual_stride) || !plain(*residual))
            return py::none();
        a.residual = residual->data_ptr();
    }
    const bool grad = wants_grad(x) || wants_grad(weight) || wants_grad(residual);
    if (grad && codes) return py::none();
    c10::DeviceGuard guard(dev);
    if (grad) {
        check_capture({x, weight, residual});
        const auto results = RmsNorm::apply(*x, *weight, residual ? std::optional<at::Tensor>(*residual) : std::nullopt, eps);
        return residual ? py::object(py::make_tuple(results[0], results[1])) : py::cast(results[0]);
    }
    const auto options = x->options().requires_grad(false).memory_format(std::nullopt);
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
    void* stream = stream_of(dev);
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
        a->numel() / K > 1 << 24 || a->numel() / K * N > (int64_t)1 << 37 || a_scales->dim() != a->dim() || a_scales->size(-1) != blocks ||
        a_scales->sizes().slice(0, a->dim() - 1) != a->sizes().slice(0, a->dim() - 1) ||
        !dims(*b_scales, {(N + 127) / 128, blocks}) || a->scalar_type() != at::kFloat8_e4m3fn ||
        b->scalar_type() != at::kFloat8_e4m3fn || a_scales->scalar_type() != at::kFloat ||
        b_scales->scalar_type() != at::kFloat)
        return py::none();
    for (const at::Tensor* t : {a, a_scales, b, b_scales})
        if (t->device() != dev || !t->is_contiguous() || !plain(*t) || wants_grad(t)) return py::none();
    p.a = static_cast<const uint8_t*>(a->data_ptr());
    p.a_scales = static_cast<const float*>(a_scales->data_ptr());
    p.b = static_cast<const uint8_t*>(b->data_ptr());
    p.b_scales = static_cast<const float*>(b_scales->data_ptr());
    if (!aligned(p.a, 16) || !aligned(p.b, 16)) return py::none();
    p.M = (int32_t)(a->numel() / K);
    p.N = (int32_t)N;
    p.K = (int32_t)K;
    c10::DeviceGuard guard(dev);
    auto shape = a->sizes().vec();
    shape.back() = N;
    const auto options = a->options().requires_grad(false).memory_format(std::nullopt);
    at::Tensor out = at::empty(shape, options.dtype(type));
    p.out = out.data_ptr();
    const int rc = g_product(&p, stream_of(dev));
    if (rc != 0) return py::int_(rc);
    return py::cast(out);
}

// The same check for the Python path, of tensors or None.
void capturable(py::handle x, py::handle weight, py::handle residual) {
    const at::Tensor* t = tensor(x);
    c10::DeviceGuard guard(t->device());
    check_capture({t, tensor(weight), tensor(residual)});
}

void set_entry(uint64_t norm_address, uint64_t norm_fp8, uint64_t product, uint64_t grad_bytes, uint64_t grad,
               uint64_t error) {
    g_norm = reinterpret_cast<decltype(g_norm)>(norm_address);
    g_norm_fp8 = reinterpret_cast<decltype(g_norm_fp8)>(norm_fp8);
    g_product = reinterpret_cast<decltype(g_product)>(product);
    g_grad_bytes = reinterpret_cast<decltype(g_grad_bytes)>(grad_bytes);
    g_grad = reinterpret_cast<decltype(g_grad)>(grad);
    g_error = reinterpret_cast<decltype(g_error)>(error);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("rms_norm", &rms_norm, "dsa_amd.rms_norm, or None");
    m.def("rms_norm_fp8", &rms_norm_fp8, "dsa_amd.rms_norm_fp8, or None");
    m.def("quantize_fp8", &quantize_fp8, "dsa_amd.quantize_fp8, or None");
    m.def("matmul_fp8", &matmul_fp8, "dsa_amd.matmul_fp8, or None");
    m.def("capturable", &capturable, "raises where the gradient of these cannot be captured now");
    m.def("set_entry", &set_entry, "addresses of the library's entry points");
}
