// Host fast path of dsa_amd.extend_block_table, rotary, write_kv_rows and
// forward_shared (no reference counterpart: the reference takes its cache as
// given, dsa/api.py:30-33).
//
// A decode step's kernels take 3 to 4 us (forward_shared's 20), their checks,
// output and launch in Python 9 to 10 (15).  Here the same work takes 3 to 6.
// Nothing is raised for a bad input: whatever the Python path would reject, and
// what it does besides (a gradient or tangent to record, nothing to do), returns
// None, and the caller goes on in Python.  A failed launch returns the library's status code.  Nothing is
// allocated or launched before every check has passed.
#include <torch/extension.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <utility>

#include "dsa_mi355x_cache.h"

namespace {

decltype(&dsa_extend_block_table) g_extend = nullptr;
decltype(&dsa_rotary) g_rotary = nullptr;
decltype(&dsa_write_kv_rows) g_write = nullptr;
decltype(&dsa_fwd_shared_ws_bytes) g_shared_bytes = nullptr;
decltype(&dsa_fwd_shared) g_shared = nullptr;

const at::Tensor* tensor(py::handle h) { return THPVariable_Check(h.ptr()) ? &THPVariable_Unpack(h.ptr()) : nullptr; }

// An int of exactly that type in [low, high].
bool integer(py::handle h, int64_t low, int64_t high, int64_t& value) {
    if (!PyLong_CheckExact(h.ptr())) return false;
    int overflow = 0;
    value = PyLong_AsLongLongAndOverflow(h.ptr(), &overflow);
    return overflow == 0 && value >= low && value <= high;
}

bool flag(py::handle h, bool& value) {
    if (!PyBool_Check(h.ptr())) return false;
    value = h.ptr() == Py_True;
    return true;
}

bool magnitude_of(py::handle h, float& value) {
    if (!PyFloat_CheckExact(h.ptr())) return false;
    const double d = PyFloat_AS_DOUBLE(h.ptr());
    if (!(std::abs(d) <= 3.4028234663852886e38)) return false;
    value = (float)d;
    return true;
}

bool vector(const at::Tensor* t, at::ScalarType type, c10::Device dev, int64_t size) {
    return t && t->dim() == 1 && (size < 0 || t->size(0) == size) && t->scalar_type() == type && t->device() == dev &&
           t->is_contiguous();
}

bool frequencies_ok(const at::Tensor* t, c10::Device dev) {
    return vector(t, at::kDouble, dev, -1) && t->size(0) >= 1 && t->size(0) <= DSA_ROTARY_MAX_DIM / 2;
}

bool positions_ok(const at::Tensor* t, c10::Device dev) {
    return t && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->device() == dev &&
           t->is_contiguous();
}

bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Autograd is told of a tensor that a call writes in place.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Whether it carries a forward-mode derivative, or is one of a function transform's stand-ins (they hold no memory).
bool differentiated(const at::Tensor& t) { return t._fw_grad(0).defined() || !t.has_storage(); }

// No two elements share memory: each dimension steps over the ones inside it.
bool distinct(const at::Tensor& t) {
    std::array<std::pair<int64_t, int64_t>, 4> steps;
    int n = 0;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) steps[n++] = {t.stride(i), t.size(i)};
    std::sort(steps.begin(), steps.begin() + n);
    int64_t reach = 1;
    for (int i = 0; i < n; ++i) {
        if (steps[i].first < reach) return false;
        reach += (steps[i].second - 1) * steps[i].first;
    }
    return true;
}

// Addresses [first, last) of a tensor's elements.
std::pair<uintptr_t, uintptr_t> span(const at::Tensor& t) {
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
    return {p, p + last * t.element_size()};
}

py::object extend_block_table(py::handle htable, py::handle hlengths, py::handle hnew, py::handle hfree,
                              py::handle hblock, py::handle hmax) {
    const at::Tensor *table = tensor(htable), *lengths = tensor(hlengths), *fresh = tensor(hnew), *free = tensor(hfree);
    int64_t block, tokens;
    if (!table || table->dim() != 2 || !integer(hblock, 1, 0x7fffffff, block) || !integer(hmax, 0, 0x7fffffff, tokens))
        return py::none();
    const int64_t B = table->size(0), columns = table->size(1);
    const c10::Device dev = table->device();
    if (B < 1 || B > DSA_TABLE_MAX_SEQUENCES || columns < 1 || columns > 0x7fffffff || !dev.is_cuda() ||
        !table->is_contiguous() || table->scalar_type() != at::kInt || !vector(lengths, at::kInt, dev, B) ||
        !vector(fresh, at::kInt, dev, B) || !vector(free, at::kInt, dev, -1) || free->size(0) > 0x7fffffff)
        return py::none();
    c10::DeviceGuard guard(dev);
    at::Tensor all = at::empty({2 * tokens + 2 * B + 2}, table->options().requires_grad(false));
    int32_t* p = static_cast<int32_t*>(all.data_ptr());
    const int rc = g_extend(static_cast<int32_t*>(table->data_ptr()), static_cast<const int32_t*>(lengths->data_ptr()),
                            static_cast<const int32_t*>(fresh->data_ptr()), static_cast<const int32_t*>(free->data_ptr()),
                            p, p + tokens, p + 2 * tokens, p + 2 * tokens + B + 1, p + 2 * tokens + 2 * B + 1, (int)B,
                            (int)columns, (int)block, (int)free->size(0), (int)tokens,
                            c10::hip::getCurrentHIPStream(dev.index()).stream());
    if (rc != 0) return py::int_(rc);
    written(*table);
    at::AutoDispatchBelowADInplaceOrView plain;  // views of whole numbers: nothing to record
    return py::make_tuple(all.narrow(0, 0, tokens), all.narrow(0, tokens, tokens), all.narrow(0, 2 * tokens, B + 1),
                          all.narrow(0, 2 * tokens + B + 1, B), all.narrow(0, 2 * tokens + 2 * B + 1, 1));
}

py::object rotary(py::handle hx, py::handle hpositions, py::handle hfrequencies, py::handle hinterleaved,
                  py::handle hstart, py::handle htransposed, py::handle hmagnitude, py::handle hout) {
    const at::Tensor *x = tensor(hx), *positions = tensor(hpositions), *frequencies = tensor(hfrequencies);
    const at::Tensor* out = tensor(hout);
    bool interleaved, transposed;
    dsa_rotary_args a{};
    int64_t start;
    if (!x || (!out && !hout.is_none()) || (x->dim() != 3 && x->dim() != 4) || x->numel() == 0 ||
        !flag(hinterleaved, interleaved) || !flag(htransposed, transposed) || !magnitude_of(hmagnitude, a.magnitude))
        return py::none();
    const c10::Device dev = x->device();
    const auto type = x->scalar_type();
    const int64_t n = x->dim(), width = x->size(n - 1);
    if (!dev.is_cuda() || (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat) ||
        !frequencies_ok(frequencies, dev) || !positions_ok(positions, dev) ||
        positions->sizes() != x->sizes().slice(0, n - 2) || width > 0x7fffffff || x->size(n - 2) > 0x7fffffff ||
        !integer(hstart, 0, width - 2 * frequencies->size(0), start) || x->stride(n - 1) != 1)
        return py::none();
    if (at::GradMode::is_enabled() &&
        (x->requires_grad() || frequencies->requires_grad() || (out && out->requires_grad())))
        return py::none();
    if (differentiated(*x) || (out && differentiated(*out)) || differentiated(*frequencies) || !positions->has_storage())
        return py::none();
    if (out) {
        if (out->sizes() != x->sizes() || out->scalar_type() != type || out->device() != dev || out->stride(n - 1) != 1 ||
            !distinct(*out))
            return py::none();
        if (out->data_ptr() != x->data_ptr() || out->strides() != x->strides()) {
            const auto xs = span(*x), ys = span(*out);
            if (xs.first < ys.second && ys.first < xs.second) return py::none();
        }
    }
    c10::DeviceGuard guard(dev);
    at::Tensor fresh;
    if (!out) {
        fresh = at::empty(x->sizes(), x->options().requires_grad(false));
        out = &fresh;
    }
    a.x = x->data_ptr();
    a.out = out->data_ptr();
    a.positions = positions->data_ptr();
    a.frequencies = static_cast<const double*>(frequencies->data_ptr());
    a.groups = n == 4 ? x->size(0) : 1;
    a.tokens = x->size(n - 3);
    for (int i = 0; i < 3; ++i) {
        a.x_stride[i] = i > 0 || n == 4 ? x->stride(n - 4 + i) : 0;
        a.out_stride[i] = i > 0 || n == 4 ? out->stride(n - 4 + i) : 0;
    }
    a.heads = (int32_t)x->size(n - 2);
    a.width = (int32_t)width;
    a.start = (int32_t)start;
    a.dim = (int32_t)(2 * frequencies->size(0));
    a.dtype = type == at::kBFloat16 ? DSA_BF16 : type == at::kHalf ? DSA_F16 : DSA_F32;
    a.positions_64 = positions->scalar_type() == at::kLong;
    a.interleaved = interleaved;
    a.transposed = transposed;
    const int rc = g_rotary(&a, c10::hip::getCurrentHIPStream(dev.index()).stream());
    if (rc != 0) return py::int_(rc);
    if (!fresh.defined()) written(*out);
    return fresh.defined() ? py::cast(fresh) : py::reinterpret_borrow<py::object>(hout);
}

py::object write_kv_rows(py::handle hkv, py::handle hrope, py::handle hslots, py::handle hcache, py::handle hrope_cache,
                         py::handle hpositions, py::handle hfrequencies, py::handle hinterleaved, py::handle hmagnitude,
                         py::handle hpow2) {
    const at::Tensor *kv = tensor(hkv), *rope = tensor(hrope), *slots = tensor(hslots), *cache = tensor(hcache);
    const at::Tensor *rope_cache = tensor(hrope_cache), *positions = tensor(hpositions);
    const at::Tensor* frequencies = tensor(hfrequencies);
    bool interleaved, pow2;
    dsa_write_args a{};
    if (!kv || !rope || !cache || (!rope_cache && !hrope_cache.is_none()) || (!positions && !hpositions.is_none()) ||
        (!frequencies && !hfrequencies.is_none()) || !positions != !frequencies || !flag(hinterleaved, interleaved) ||
        !flag(hpow2, pow2) || !magnitude_of(hmagnitude, a.magnitude) || kv->dim() != 2 || rope->dim() != 2 ||
        cache->dim() < 2)
        return py::none();
    const int64_t tokens = kv->size(0);
    const c10::Device dev = kv->device();
    const bool fp8 = cache->scalar_type() == at::kByte;
    const auto bf16 = at::kBFloat16;
    if (tokens == 0 || cache->numel() == 0 || kv->size(1) != 512 || rope->size(0) != tokens || rope->size(1) != 64 ||
        !dev.is_cuda() || rope->device() != dev || cache->device() != dev || !cache->is_contiguous() ||
        cache->size(-1) != (fp8 ? 656 : 512) || kv->scalar_type() != bf16 || rope->scalar_type() != bf16 ||
        !vector(slots, at::kInt, dev, tokens) || fp8 != !rope_cache)
        return py::none();
    const int64_t rows = cache->numel() / cache->size(-1);
    if (!fp8) {
        const int64_t n = cache->dim();
        if (cache->scalar_type() != bf16 || rope_cache->scalar_type() != bf16 || rope_cache->device() != dev ||
            !rope_cache->is_contiguous() || rope_cache->dim() != n || rope_cache->size(n - 1) != 64 ||
            rope_cache->sizes().slice(0, n - 1) != cache->sizes().slice(0, n - 1))
            return py::none();
        if (at::GradMode::is_enabled() && (cache->requires_grad() || rope_cache->requires_grad())) return py::none();
        if (differentiated(*cache) || differentiated(*rope_cache)) return py::none();
        a.rope_cache = static_cast<uint16_t*>(rope_cache->data_ptr());
    }
    if (frequencies) {
        if (!frequencies_ok(frequencies, dev) || frequencies->size(0) != 32 || !positions_ok(positions, dev) ||
            positions->dim() != 1 || positions->size(0) != tokens)
            return py::none();
        a.positions = positions->data_ptr();
        a.frequencies = static_cast<const double*>(frequencies->data_ptr());
        a.positions_64 = positions->scalar_type() == at::kLong;
    }
    if (kv->stride(1) != 1 || rope->stride(1) != 1 || (tokens > 1 && (kv->stride(0) % 8 || rope->stride(0) % 2)) ||
        !aligned(kv->data_ptr(), 16) || !aligned(rope->data_ptr(), 4) || !aligned(cache->data_ptr(), 16) ||
        !aligned(a.rope_cache, 4))
        return py::none();
    c10::DeviceGuard guard(dev);
    a.kv = static_cast<const uint16_t*>(kv->data_ptr());
    a.k_rope = static_cast<const uint16_t*>(rope->data_ptr());
    a.slots = static_cast<const int32_t*>(slots->data_ptr());
    a.cache = cache->data_ptr();
    a.tokens = tokens;
    a.cache_rows = rows;
    a.kv_stride = tokens > 1 ? kv->stride(0) : 512;
    a.rope_stride = tokens > 1 ? rope->stride(0) : 64;
    a.kv_format = fp8 ? 1 : 0;
    a.pow2_scales = pow2;
    a.interleaved = interleaved;
    const int rc = g_write(&a, c10::hip::getCurrentHIPStream(dev.index()).stream());
    if (rc == 0) {
        written(*cache);
        if (rope_cache) written(*rope_cache);
    }
    return py::int_(rc);
}

bool dims(const at::Tensor& t, std::initializer_list<int64_t> want) {
    return t.sizes() == at::IntArrayRef(want.begin(), want.size());
}

py::object forward_shared(py::handle hq, py::handle hkv, py::handle hq_rope, py::handle hk_rope, py::handle hlengths,
                          py::handle hprefix, py::handle hscale, py::handle htable) {
    const at::Tensor *q = tensor(hq), *kv = tensor(hkv), *q_rope = tensor(hq_rope), *k_rope = tensor(hk_rope);
    const at::Tensor *lengths = tensor(hlengths), *table = tensor(htable);
    if (!q || !kv || !q_rope || !lengths || (!k_rope && !hk_rope.is_none()) || (!table && !htable.is_none()) ||
        q->dim() != 4 || kv->dim() != 4)
        return py::none();
    const bool fp8 = kv->scalar_type() == at::kByte;
    const auto bf16 = at::kBFloat16;
    const int64_t B = q->size(0), SQ = q->size(1), H = q->size(2);
    int64_t n = B, rows = kv->size(1), L = rows, prefix;  // kv [n, rows, 1, ..]
    dsa_shared_args a{};
    const c10::Device dev = q->device();
    if (!dev.is_cuda()) return py::none();
    if (table) {
        if (table->dim() != 2 || table->size(0) != B || table->scalar_type() != at::kInt || table->device() != dev ||
            !table->is_contiguous())
            return py::none();
        n = kv->size(0);
        if (n <= 0 || rows <= 0 || n > 1 << 25 || rows > 1 << 25 || table->size(1) > 1 << 25) return py::none();
        L = table->size(1) * rows;
        a.block_table = static_cast<const int32_t*>(table->data_ptr());
        a.block_size = (int32_t)rows;
        a.max_blocks = (int32_t)table->size(1);
        a.num_blocks = (int32_t)n;
    }
    if (fp8 != !k_rope || B <= 0 || SQ <= 0 || H <= 0 || L <= 0 || L >= 1 << 25 || B > 1 << 30 || SQ > 1 << 30 ||
        H > 1 << 30 || !dims(*q, {B, SQ, H, 512}) || !dims(*q_rope, {B, SQ, H, 64}) || !dims(*lengths, {B, SQ}) ||
        !dims(*kv, {n, rows, 1, fp8 ? 656 : 512}) || (!fp8 && !dims(*k_rope, {n, rows, 1, 64})) ||
        q->scalar_type() != bf16 || q_rope->scalar_type() != bf16 || lengths->scalar_type() != at::kInt ||
        (!fp8 && (kv->scalar_type() != bf16 || k_rope->scalar_type() != bf16)) || !integer(hprefix, 0, L, prefix))
        return py::none();
    for (const at::Tensor* t : {q, kv, q_rope, lengths, fp8 ? q : k_rope})
        if (t->device() != dev || !t->is_contiguous()) return py::none();
    if (!hscale.is_none()) {
        if (!PyFloat_CheckExact(hscale.ptr())) return py::none();
        a.scale = (float)PyFloat_AS_DOUBLE(hscale.ptr());
        if (!(a.scale > 0.f) || !std::isfinite(a.scale)) return py::none();
    }
    a.B = (int32_t)B;
    a.SQ = (int32_t)SQ;
    a.H = (int32_t)H;
    a.L = (int32_t)L;
    a.prefix = (int32_t)prefix;
    a.kv_format = fp8 ? 1 : 0;
    a.q = static_cast<const uint16_t*>(q->data_ptr());
    a.kv = kv->data_ptr();
    a.q_rope = static_cast<const uint16_t*>(q_rope->data_ptr());
    a.k_rope = fp8 ? nullptr : static_cast<const uint16_t*>(k_rope->data_ptr());
    a.lengths = static_cast<const int32_t*>(lengths->data_ptr());
    for (const void* p : {(const void*)a.q, a.kv, (const void*)a.q_rope, (const void*)a.k_rope})
        if (!aligned(p, 16)) return py::none();
    c10::DeviceGuard guard(dev);
    a.workspace_bytes = g_shared_bytes(&a);
    if (a.workspace_bytes < 0) return py::none();
    const auto options = q->options().requires_grad(false);
    at::Tensor out = at::empty(q->sizes(), options);
    at::Tensor top = at::empty({B, 1, SQ, H}, options.dtype(at::kFloat)), sum = at::empty_like(top);
    at::Tensor workspace = at::empty({a.workspace_bytes}, options.dtype(at::kByte));
    a.out = static_cast<uint16_t*>(out.data_ptr());
    a.out_max = static_cast<float*>(top.data_ptr());
    a.out_sum = static_cast<float*>(sum.data_ptr());
    a.workspace = workspace.data_ptr();
    const int rc = g_shared(&a, c10::hip::getCurrentHIPStream(dev.index()).stream());
    if (rc != 0) return py::int_(rc);
    return py::make_tuple(out, top, sum);
}

void set_entry(uint64_t extend, uint64_t rotary_address, uint64_t write, uint64_t shared_bytes, uint64_t shared) {
    g_extend = reinterpret_cast<decltype(g_extend)>(extend);
    g_rotary = reinterpret_cast<decltype(g_rotary)>(rotary_address);
    g_write = reinterpret_cast<decltype(g_write)>(write);
    g_shared_bytes = reinterpret_cast<decltype(g_shared_bytes)>(shared_bytes);
    g_shared = reinterpret_cast<decltype(g_shared)>(shared);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("extend_block_table", &extend_block_table, "dsa_amd.extend_block_table, or None");
    m.def("rotary", &rotary, "dsa_amd.rotary, or None");
    m.def("write_kv_rows", &write_kv_rows, "dsa_amd.write_kv_rows (0), or None");
    m.def("forward_shared", &forward_shared, "dsa_amd.forward_shared, or None");
    m.def("set_entry", &set_entry, "addresses of the library's entry points");
}
