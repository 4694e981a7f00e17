// Host half of the training operators (geneface_amd.optim, geneface_amd.fp8): takes torch tensors, checks them and calls the C ABI of
// libgeneface_hip.so (include/geneface_train_hip.h), whose functions are handed over once as addresses (bind), so that both halves are of one library.
//
// A step over a few dozen small tensors takes the GPU five microseconds; asking each tensor in Python for its type, size, device, layout and
// address took fifty, and a layer's forward and backward call in Python seventy more than its launches.  This module does the same in C++.
#include <ATen/autocast_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstring>
#include <deque>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "geneface_train_hip.h"

namespace {

namespace py = pybind11;
using at::Tensor;

// The tensors of a Python list or tuple where they lie in their Python objects, which the sequence holds as long as the call takes.  A vector of tensors
// would count every one's references up and down again: 24 tensors of 32 bits take 8.0 us so, 10.3 that way; 200 take 36 for 57.
struct Tensors {
    py::object sequence;
    std::vector<const Tensor*> at;
    std::deque<Tensor> own;      // those that replace one of the caller's

    explicit Tensors(const py::object& given) : sequence(py::reinterpret_steal<py::object>(PySequence_Fast(given.ptr(), "a list of tensors is needed"))) {
        if (!sequence) throw py::error_already_set();
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(sequence.ptr());
        PyObject** items = PySequence_Fast_ITEMS(sequence.ptr());
        at.reserve(n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (!THPVariable_Check(items[i])) throw py::type_error("a list of tensors is needed");
            at.push_back(&THPVariable_Unpack(items[i]));
        }
    }
    size_t size() const { return at.size(); }
    const Tensor& operator[](size_t i) const { return *at[i]; }
    void replace(size_t i, Tensor t) {
        own.push_back(std::move(t));
        at[i] = &own.back();
    }
};

struct Api {
    int (*adamw_step)(const gf_adamw_t*, void*);
    uint64_t (*grad_norm_workspace_bytes)(uint32_t);
    int (*grad_norm)(const gf_grad_norm_t*, void*);
    int (*linear_plan)(gf_fp8_linear_t*);
    int (*linear)(const gf_fp8_linear_t*, void*);
    int (*linear_backward)(const gf_fp8_linear_backward_t*, void*);
    const char* (*last_error)(void);
} api;

void bind(const std::vector<uint64_t>& a) {
    if (a.size() != sizeof(api) / 8) throw std::runtime_error("bind: wrong number of functions");
    memcpy(&api, a.data(), sizeof(api));
}

void check(int rc) {
    if (rc) throw std::runtime_error(api.last_error());
}

void refuse_unless(bool ok, const char* message) {
    if (!ok) throw std::runtime_error(message);
}

std::string name_of(at::ScalarType t) { return std::string("torch.") + c10::toString(t); }

std::string name_of(const at::Device& d) { return d.str(); }

std::string name_of(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += std::to_string(s[i]) + (i + 1 < s.size() ? ", " : s.size() == 1 ? "," : "");
    return r + ")";
}

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return GF_F32;
        case at::kBFloat16: return GF_BF16;
        case at::kHalf: return GF_F16;
        default: return -1;
    }
}

void* stream_of(const at::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

void same_device(const char* what, const Tensors& list, const at::Device& d) {
    if (d.type() != at::kCUDA) throw std::runtime_error(std::string(what) + " must be CUDA tensors");
    for (const Tensor* t : list.at)
        if (t->device() != d) throw std::runtime_error(std::string(what) + " must all be on " + name_of(d));
}

void strided(const char* what, const Tensors& list) {
    for (const Tensor* t : list.at)
        if (t->layout() != at::kStrided) throw std::runtime_error(std::string(what) + ": sparse gradients are not supported");
}

// t as its memory has to be: consecutive values, no sign left to be applied (a view such as conj().imag carries one)
Tensor plain(const Tensor& t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }

// Address of one float32 on the device, or NULL.
const float* scalar(const char* name, const std::optional<Tensor>& t, const at::Device& d) {
    if (!t) return nullptr;
    if (t->scalar_type() != at::kFloat || t->layout() != at::kStrided || t->numel() != 1 || t->device() != d)
        throw std::runtime_error(std::string(name) + " must be one float32 value on " + name_of(d));
    return static_cast<const float*>(t->data_ptr());
}

struct Span { uintptr_t first, behind; };      // bytes from first to behind

// By bytes of the address that differ among them, lowest first: 96 spans (24 tensors) take 1.4 us, 3.1 by comparisons.
void sort_by_address(std::vector<Span>& spans) {
    if (spans.size() < 32) {
        std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
        return;
    }
    uintptr_t differ = 0;
    for (const Span& s : spans) differ |= s.first ^ spans[0].first;
    std::vector<Span> other(spans.size());
    for (int shift = 0; shift < 64; shift += 8) {
        if (!(differ >> shift & 255)) continue;
        uint32_t at[256] = {}, sum = 0;
        for (const Span& s : spans) ++at[s.first >> shift & 255];
        for (uint32_t& a : at) {
            const uint32_t here = a;
            a = sum;
            sum += here;
        }
        for (const Span& s : spans) other[at[s.first >> shift & 255]++] = s;
        spans.swap(other);
    }
}

// Whether anything of [first, behind) is among the sorted spans, which do not overlap.
bool touches(const std::vector<Span>& spans, uintptr_t first, uintptr_t behind) {
    const auto next = std::upper_bound(spans.begin(), spans.end(), first, [](uintptr_t a, const Span& s) { return a < s.behind; });      // the first that ends behind `first`
    return next != spans.end() && next->first < behind;
}

// ---- AdamW ---------------------------------------------------------------------------------------------------------------------------------

void adamw_step(const py::object& params_, const py::object& grads_, const py::object& m_, const py::object& v_, const py::object& steps_, double lr,
                const std::optional<Tensor>& lr_device, double beta1, double beta2, double eps, double weight_decay, const py::object& m_scales_, const py::object& v_scales_,
                const std::optional<Tensor>& grad_scale, const std::optional<Tensor>& found_inf, const std::optional<Tensor>& grad_norm, const std::optional<Tensor>& grad_norm_wide,
                double max_norm) {
    const Tensors params(params_), m(m_), v(v_), steps(steps_);
    Tensors grads(grads_);
    std::optional<Tensors> m_scales, v_scales;
    if (!m_scales_.is_none()) { m_scales.emplace(m_scales_); v_scales.emplace(v_scales_); }
    const bool eight = m_scales.has_value();
    const size_t n = params.size();
    for (const Tensors* l : {(const Tensors*)&grads, &m, &v, &steps, eight ? &*m_scales : &m, eight ? &*v_scales : &v})
        refuse_unless(l->size() == n, "adamw_step: lists of unlike lengths");
    if (!n) return;
    strided("adamw_step", grads);
    const at::Device dev = params[0].device();
    bool kinds[3] = {false, false, false};
    for (size_t i = 0; i < n; ++i) {
        const int64_t size = params[i].numel();
        const int kind = dtype_of(params[i]);
        refuse_unless(grads[i].scalar_type() == params[i].scalar_type(), "adamw_step: a gradient must have its parameter's dtype");
        refuse_unless(kind >= 0, "adamw_step: parameters must be float32, bfloat16 or float16");
        kinds[kind] = true;
        refuse_unless(grads[i].numel() == size && m[i].numel() == size && v[i].numel() == size, "adamw_step: gradients and moments must have their parameter's size");
        const at::ScalarType state = eight ? at::kFloat8_e4m3fn : at::kFloat;
        refuse_unless(m[i].scalar_type() == state && v[i].scalar_type() == state,
                      eight ? "adamw_step: moments must be torch.float8_e4m3fn with scales" : "adamw_step: moments must be torch.float32 without scales");
        refuse_unless(steps[i].scalar_type() == at::kFloat && steps[i].numel() == 1, "adamw_step: each step must be one float32 value");
        if (eight) {
            const int64_t blocks = (size + 127) / 128;
            for (const Tensors* l : {&*m_scales, &*v_scales})
                refuse_unless((*l)[i].scalar_type() == at::kFloat && (*l)[i].numel() == blocks, "adamw_step: scales must be float32 with one value for each 128 of the parameter");
        }
    }
    const char* all = "adamw_step: all tensors";
    same_device(all, params, dev);
    same_device(all, grads, dev);
    for (const Tensors* l : {&m, &v, &steps}) same_device(all, *l, dev);
    if (eight) { same_device(all, *m_scales, dev); same_device(all, *v_scales, dev); }
    const c10::OptionalDeviceGuard guard(dev);
    std::vector<Span> written;      // what the step writes, each value once
    written.reserve(6 * n);
    auto writes = [&](const Tensor& t) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
        written.push_back({at, at + t.nbytes()});
    };
    for (size_t i = 0; i < n; ++i) {
        const bool dense = params[i].is_contiguous() && !params[i].is_neg() && m[i].is_contiguous() && v[i].is_contiguous() && (!eight || ((*m_scales)[i].is_contiguous() && (*v_scales)[i].is_contiguous()));
        refuse_unless(dense, "adamw_step: parameters and their state must be contiguous tensors");
        if (!grads[i].is_contiguous() || grads[i].is_neg()) grads.replace(i, plain(grads[i]));
        writes(steps[i]);
        if (!params[i].numel()) continue;      // (empty tensors have no address)
        writes(params[i]);
        writes(m[i]);
        writes(v[i]);
        if (eight) {
            writes((*m_scales)[i]);
            writes((*v_scales)[i]);
        }
    }
    sort_by_address(written);
    for (size_t i = 1; i < written.size(); ++i)
        refuse_unless(written[i - 1].behind <= written[i].first, "adamw_step: the same tensor is given twice, or two that share memory");
    auto reads = [&](const void* p, size_t bytes) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        refuse_unless(!bytes || !touches(written, at, at + bytes), "adamw_step: a gradient or a scalar shares memory with what the step writes");
    };
    for (size_t i = 0; i < n; ++i)      // (a gradient that is its own parameter is read where it is written, by the same thread)
        if (grads[i].data_ptr() != params[i].data_ptr()) reads(grads[i].data_ptr(), grads[i].nbytes());
    for (const std::optional<Tensor>* t : {&lr_device, &grad_scale, &found_inf, &grad_norm, &grad_norm_wide})
        if (*t) reads((*t)->data_ptr(), (*t)->nbytes());
    gf_adamw_t d = {};
    d.state_bits = eight ? 8 : 32;
    d.lr = lr; d.beta1 = beta1; d.beta2 = beta2; d.eps = eps; d.weight_decay = weight_decay; d.max_norm = max_norm;
    d.lr_device = scalar("lr", lr_device, dev);
    d.grad_scale = scalar("grad_scale", grad_scale, dev);
    d.found_inf = scalar("found_inf", found_inf, dev);
    d.grad_norm = scalar("grad_norm", grad_norm, dev);
    if (grad_norm_wide && grad_norm_wide->device() == dev && grad_norm_wide->scalar_type() == at::kDouble && grad_norm_wide->numel() == 1)
        d.grad_norm_wide = static_cast<const double*>(grad_norm_wide->data_ptr());
    std::vector<gf_adamw_tensor_t> table;
    table.reserve(n);
    for (int kind = 0; kind < 3; ++kind) {
        if (!kinds[kind]) continue;
        table.clear();
        for (size_t i = 0; i < n; ++i) {
            if (dtype_of(params[i]) != kind) continue;
            table.push_back({params[i].data_ptr(), grads[i].data_ptr(), m[i].data_ptr(), v[i].data_ptr(), eight ? (float*)(*m_scales)[i].data_ptr() : nullptr,
                             eight ? (float*)(*v_scales)[i].data_ptr() : nullptr, (float*)steps[i].data_ptr(), (uint64_t)params[i].numel()});
        }
        d.tensors_host = table.data();
        d.count = (uint32_t)table.size();
        d.dtype = kind;
        check(api.adamw_step(&d, stream_of(dev)));
    }
    // written through raw pointers: whoever keys on a tensor's version has to see it
    for (const Tensors* l : {&params, &m, &v, &steps, eight ? (const Tensors*)&*m_scales : nullptr, eight ? (const Tensors*)&*v_scales : nullptr})
        if (l)
            for (const Tensor* t : l->at)
                if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

std::pair<Tensor, Tensor> grad_norm(const py::object& grads_, const std::optional<Tensor>& grad_scale) {
    Tensors grads(grads_);
    refuse_unless(grads.size(), "grad_norm: no gradients");
    strided("grad_norm", grads);
    const at::Device dev = grads[0].device();
    for (const Tensor* g : grads.at) refuse_unless(dtype_of(*g) >= 0, "grad_norm: gradients must be float32, bfloat16 or float16");
    same_device("grad_norm: the gradients", grads, dev);
    const c10::OptionalDeviceGuard guard(dev);
    std::vector<gf_norm_tensor_t> table;
    table.reserve(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        if (!grads[i].is_contiguous() || grads[i].is_neg()) grads.replace(i, plain(grads[i]));
        table.push_back({grads[i].data_ptr(), (uint64_t)grads[i].numel(), (uint32_t)dtype_of(grads[i]), 0});
    }
    const Tensor out = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
    const Tensor work = at::empty({(int64_t)api.grad_norm_workspace_bytes((uint32_t)table.size())}, at::TensorOptions().dtype(at::kByte).device(dev));
    const Tensor wide = at::empty({}, at::TensorOptions().dtype(at::kDouble).device(dev));
    const gf_grad_norm_t d = {table.data(), (uint32_t)table.size(), 0, scalar("grad_scale", grad_scale, dev), (float*)out.data_ptr(), work.data_ptr(), (double*)wide.data_ptr()};
    check(api.grad_norm(&d, stream_of(dev)));
    return {out, wide};
}

// ---- 8-bit linear --------------------------------------------------------------------------------------------------------------------------

// t [.., K] as a matrix whose rows are consecutive values, rows at any distance
Tensor matrix(const Tensor& any) {
    const Tensor t = any.is_neg() ? any.resolve_neg() : any, m = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return m.stride(1) == 1 && m.stride(0) >= m.size(1) ? m : m.contiguous();
}

uint64_t pitch(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

at::TensorOptions bytes_on(const at::Device& d) { return at::TensorOptions().dtype(at::kByte).device(d); }

struct Product { Tensor y, saved; uint64_t backward_bytes; };

// One of weight, or codes and scales of an [n, k] weight.
Product forward(const Tensor& x_any, const Tensor* weight, const Tensor* codes, const Tensor* scales, int64_t n, bool keep_w, bool keep_x) {
    const at::Device dev = x_any.device();
    const c10::OptionalDeviceGuard guard(dev);
    const Tensor x = matrix(x_any), w = weight ? matrix(*weight) : Tensor();
    gf_fp8_linear_t d = {};
    d.x = x.data_ptr(); d.ldx = pitch(x); d.m = x.size(0); d.n = n; d.k = x.size(1); d.dtype = dtype_of(x);
    d.keep_w = keep_w; d.keep_x = keep_x;
    if (weight) { d.w = w.data_ptr(); d.ldw = pitch(w); d.w_dtype = dtype_of(w); }
    else { d.codes = (const uint8_t*)codes->data_ptr(); d.scales = (const uint8_t*)scales->data_ptr(); }
    check(api.linear_plan(&d));
    Product p;
    p.y = at::empty({x.size(0), n}, x.options());
    p.backward_bytes = d.backward_bytes;
    Tensor work;
    if (d.saved_bytes) { p.saved = at::empty({(int64_t)d.saved_bytes}, bytes_on(dev)); d.saved = p.saved.data_ptr(); }
    if (d.workspace_bytes) { work = at::empty({(int64_t)d.workspace_bytes}, bytes_on(dev)); d.workspace = work.data_ptr(); }
    d.y = p.y.data_ptr();
    check(api.linear(&d, stream_of(dev)));
    return p;
}

// Kept for the backward pass: w by columns and x by columns, in 8 bits -- neither tensor itself.
struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, bool keep_w, bool keep_x) {
        Product p = ::forward(x, &w, nullptr, nullptr, w.size(0), keep_w, keep_x);
        ctx->save_for_backward({p.saved});
        ctx->saved_data["plan"] = std::vector<int64_t>{x.size(0), x.size(1), w.size(0), (int64_t)x.scalar_type(), (int64_t)w.scalar_type(), keep_w, keep_x, (int64_t)p.backward_bytes};
        return p.y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled();      // create_graph
        const at::AutoGradMode off(false);
        const Tensor saved = ctx->get_saved_variables()[0], dy = matrix(grads[0]);
        const std::vector<int64_t> plan = ctx->saved_data["plan"].toIntVector();
        const int64_t m = plan[0], k = plan[1], n = plan[2];
        const at::Device dev = dy.device();
        const c10::OptionalDeviceGuard guard(dev);
        Tensor dx, dw;
        gf_fp8_linear_backward_t d = {};
        d.dy = dy.data_ptr(); d.lddy = pitch(dy); d.saved = saved.data_ptr(); d.m = m; d.n = n; d.k = k;
        d.keep_w = plan[5]; d.keep_x = plan[6];
        if (d.keep_w && ctx->needs_input_grad(0)) dx = at::empty({m, k}, dy.options().dtype((at::ScalarType)plan[3]));
        if (d.keep_x && ctx->needs_input_grad(1)) dw = at::empty({n, k}, dy.options().dtype((at::ScalarType)plan[4]));
        const Tensor work = at::empty({plan[7]}, bytes_on(dev));
        d.dx = dx.defined() ? dx.data_ptr() : nullptr;
        d.dw = dw.defined() ? dw.data_ptr() : nullptr;
        d.workspace = work.data_ptr();
        d.dtype = dtype_of(dy);
        d.w_dtype = dw.defined() ? dtype_of(dw) : 0;
        check(api.linear_backward(&d, stream_of(dev)));
        if (again) {
            auto error = std::make_shared<torch::autograd::DelayedError>("fp8: the gradients of linear() have no gradients of their own", 1);
            for (Tensor* t : {&dx, &dw})
                if (t->defined()) *t = (*error)({t->detach().set_requires_grad(true)})[0];
        }
        return {dx, dw, Tensor(), Tensor()};
    }
};

void check_type(const char* what, const Tensor& t) {
    if (dtype_of(t) < 0) throw std::runtime_error(std::string("fp8: ") + what + " must be float32, bfloat16 or float16, got " + name_of(t.scalar_type()));
}

Tensor checked_x(Tensor x, int64_t k, const at::Device& dev) {
    if (x.dim() < 1 || x.size(-1) != k)
        throw std::runtime_error("fp8: x of shape " + name_of(x.sizes()) + " does not fit a weight of " + std::to_string(k) + " input features");
    if (x.is_cuda() && at::autocast::is_autocast_enabled(at::kCUDA)) x = x.to(at::autocast::get_autocast_dtype(at::kCUDA));
    check_type("x", x);
    refuse_unless(x.is_cuda(), "fp8: x must be a CUDA tensor");
    if (x.device() != dev) throw std::runtime_error("fp8: x is on " + name_of(x.device()) + ", the weight on " + name_of(dev));
    return x;
}

Tensor shaped(const Tensor& y, const Tensor& x, int64_t n) {
    if (x.dim() == 2) return y;
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = n;
    return y.view(s);
}

Tensor linear(const Tensor& x_any, const Tensor& w) {
    check_type("the weight", w);
    if (w.dim() != 2) throw std::runtime_error("fp8: the weight must be a matrix, got " + name_of(w.sizes()));
    const Tensor x = checked_x(x_any, w.size(1), w.device());
    if (!x.numel() || !w.numel()) return at::matmul(x, w.t().to(x.scalar_type()));      // nothing to add up; differentiable
    const bool grad = at::GradMode::is_enabled();
    const bool keep_w = grad && x.requires_grad(), keep_x = grad && w.requires_grad();
    // (a view made inside the node could not be written in place, as a ReLU behind it does)
    return shaped(Linear::apply(x.dim() == 2 ? x : x.reshape({-1, w.size(1)}), w, keep_w, keep_x), x, w.size(0));
}

Tensor linear_packed(const Tensor& x_any, const Tensor& values, const Tensor& scales, int64_t k) {
    const Tensor x = checked_x(x_any, k, values.device());
    refuse_unless(!(at::GradMode::is_enabled() && x.requires_grad()), "fp8: an Fp8Weight has no backward pass: give the weight itself, or call under no_grad");
    const int64_t n = values.size(0);
    if (!x.numel() || !n) {
        std::vector<int64_t> s = x.sizes().vec();
        s.back() = n;
        return at::zeros(s, x.options());
    }
    return shaped(forward(x, nullptr, &values, &scales, n, false, false).y, x, n);
}

}  // namespace

PYBIND11_MODULE(_train_host, m) {
    m.def("bind", &bind);
    m.def("adamw_step", &adamw_step);
    m.def("grad_norm", &grad_norm);
    m.def("linear", &linear);
    m.def("linear_packed", &linear_packed);
}
